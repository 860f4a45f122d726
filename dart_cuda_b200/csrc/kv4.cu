// A paged k/v history held in 4 bits, and the AFT-full decode step over it.
//
// History: pages of page_size positions, each [D/W][page_size][5W/4] bytes
// (W, the slab width, is the largest of 256, 128, 64, 32 that divides D).  The
// record of a slab's W channels at one position holds, per 8 channels, 4
// bytes of k codes and 4 of v codes (channel j in bits 4j..4j+3), then per
// group of 32 channels four bf16: k step, k low, v step, v low.  A code c
// stands for low + step * c: 5 bits a value instead of 32, and a lane's 8
// channels are one 8-byte word.
//
// Quantisation of a group (k and v apart): low is the largest bf16 <= min x,
// step the smallest bf16 >= (max x - low) / 15, so that 0..15 cover the group
// whatever its offset, and code = floor((x - low) / step + 1/2), decided
// exactly: x >= low + step (c + 1/2) holds in real numbers iff it holds
// against that border rounded up to fp32 (x is an fp32 number).  |x - value|
// <= step / 2.  A group with a value that is not finite (or above 1e37 in
// magnitude) is stored with a NaN step: all its channels read as NaN.
//
// The decode step is dc_aft_decode's row t of AFT-full
// (native/src/kernels/attention.cuh:6-40),
//
//   Z[b,c] = sigmoid(q[b,c]) * sum_{i<=t} e^{k_i[c] + w[t,i]} v_i[c] / sum_{i<=t} e^{k_i[c] + w[t,i]},
//
// with t = pos[b] of its own for every sequence and the rows found through a
// block table.  The reference recomputes the whole context per token
// (example/bin/shakespear4.dart:176-214) and keeps no history.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "dc_internal.h"
#include "dc_ptx.cuh"

namespace dc {
namespace kv4 {

constexpr float kBig = 1e37f;        // larger magnitudes count as not finite
constexpr int DC_DEVERR_FULL = 0x40;  // a position past the capacity
constexpr int DC_DEVERR_PAGE = 0x200; // a slot or page id outside the pool
constexpr float kLog2e = 1.4426950408889634f;

static int slab_width(int D)
{
    for (int w = 256; w >= 32; w /= 2)
        if (D % w == 0) return w;
    return 0;
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&x)[8])
{
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16 *p, float (&x)[8])
{
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = __uint_as_float(u[j] << 16);
        x[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8<float>(float *p, const float (&x)[8])
{
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16 *p, const float (&x)[8])
{
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t *>(&h);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Pairs of fp32 numbers in a 64-bit register (the type that keeps a pair of
// equal numbers in place: float2 operands were copied at every use).
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float x, float y)
{
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 a)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c)
{
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b)
{
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b)
{
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// a * b + c rounded up
__device__ __forceinline__ f32x2 fma2_ru(f32x2 a, f32x2 b, f32x2 c)
{
    f32x2 r;
    asm("fma.rp.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Largest / smallest of three (NaN if one is, respectively ignoring NaN).
__device__ __forceinline__ float max3_nan(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float min3(float a, float b, float c)
{
    float r;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// One group's quantisation by the 4 lanes (xor 1, 2) that hold its 32 values:
// step and low (bf16 values, the same on the 4 lanes), this lane's 8 codes,
// as numbers in c and packed.  `lanes`: the lanes that take part, whole
// groups.  x is scratch.
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], float &step, float &low, float (&c)[8],
                                              uint32_t lanes = 0xffffffffu)
{
    float mx = max3_nan(max3_nan(x[0], x[1], x[2]), max3_nan(x[3], x[4], x[5]), max3_nan(x[6], x[7], x[7]));
    float mn = min3(min3(x[0], x[1], x[2]), min3(x[3], x[4], x[5]), min3(x[6], x[7], x[7]));
#pragma unroll
    for (int o = 1; o <= 2; o *= 2) {
        const float other = __shfl_xor_sync(lanes, mx, o);
        mx = max3_nan(mx, other, other);
        mn = fminf(mn, __shfl_xor_sync(lanes, mn, o));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = 0.f;
    if (!(mx <= kBig && mn >= -kBig)) {
        step = __uint_as_float(0x7fff0000u);
        low = 0.f;
        return 0;
    }
    uint32_t cut = __float_as_uint(mn) & 0xffff0000u;  // towards zero
    if (__uint_as_float(cut) > mn) cut += 0x10000u;
    low = __uint_as_float(cut == 0x80000000u ? 0u : cut);  // -0 is stored as 0
    // the smallest bf16 whose 15-fold (exact in fp32) is not below mx - low
    // (then not below that rounded up): the estimate is at most one off
    const float range = fabsf(__fsub_ru(mx, low));
    uint32_t s = (__float_as_uint(range * (1.f / 15.f)) + 0xffffu) & 0xffff0000u;
    if (15.f * __uint_as_float(s) < range)
        s += 0x10000u;
    else if (s && 15.f * __uint_as_float(s - 0x10000u) >= range)
        s -= 0x10000u;
    step = __uint_as_float(s);
    if (step == 0.f) return 0;
    float st = step, lo = low;
    if (step < 1e-30f) {  // then every value is small enough to scale, exactly
        st *= 0x1p100f;
        lo *= 0x1p100f;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= 0x1p100f;
    }
    // (x - low) / step is off by at most 2^-21 of its value, so the nearest
    // whole number is the code unless that lies 0.5 away to within 1e-5 (as
    // often with bf16 values); then the border between the two decides
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(st));
    const f32x2 inv2 = pack2(inv, inv), lo2 = pack2(lo, lo);
    float2 r[4];
    float worst = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f32x2 d = add2(pack2(x[2 * j], x[2 * j + 1]), lo2 ^ 0x8000000080000000ull);
        const f32x2 k = add2(fma2(d, inv2, pack2(12582912.f, 12582912.f)), pack2(-12582912.f, -12582912.f));
        r[j] = unpack2(fma2(d, inv2, k ^ 0x8000000080000000ull));
        worst = fmaxf(worst, fmaxf(fabsf(r[j].x), fabsf(r[j].y)));
        c[2 * j] = unpack2(k).x;
        c[2 * j + 1] = unpack2(k).y;
    }
    if (worst > 0.49999f) {
        const f32x2 st2 = pack2(st, st);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x2 half = pack2(copysignf(0.5f, r[j].x), copysignf(0.5f, r[j].y));
            const f32x2 border = add2(pack2(c[2 * j], c[2 * j + 1]), half);
            const float2 y = unpack2(fma2_ru(st2, border, lo2));
            const f32x2 side = pack2(x[2 * j] >= y.x ? 0.5f : -0.5f, x[2 * j + 1] >= y.y ? 0.5f : -0.5f);
            const float2 k = unpack2(add2(border, side));
            c[2 * j] = k.x;
            c[2 * j + 1] = k.y;
        }
    }
    // four codes are the digits of a number below 2^16
    const float lo4 = fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]) + 8388608.f;
    const float hi4 = fmaf(fmaf(fmaf(c[7], 16.f, c[6]), 16.f, c[5]), 16.f, c[4]) + 8388608.f;
    return __byte_perm(__float_as_uint(lo4), __float_as_uint(hi4), 0x5410);
}

__device__ __forceinline__ uint32_t pack_params(float step, float low)
{
    return (__float_as_uint(step) >> 16) | (__float_as_uint(low) & 0xffff0000u);
}

// The 8 values that codes stand for.
__device__ __forceinline__ void values8(uint32_t codes, uint32_t params, double (&x)[8])
{
    const double step = __uint_as_float(params << 16), low = __uint_as_float(params & 0xffff0000u);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fma(step, (double)((codes >> (4 * j)) & 15u), low);
}

// Two codes as fp32 numbers 1/2 + c/32: the codes of a word are masked into
// bits 3..6 of its bytes (8 codes: two words, of even and odd channels), and
// a byte becomes the top of a mantissa by one byte permutation.  Pair j holds
// channels 0, 2 | 4, 6 | 1, 3 | 5, 7.
__device__ __forceinline__ f32x2 factors(uint32_t even, uint32_t odd, int j)
{
    const uint32_t w = j < 2 ? even : odd;
    const uint32_t k = 2 * (j & 1);
    return pack2(__uint_as_float(__byte_perm(w, 0x3f000000u, 0x7044u | k << 8)),
                 __uint_as_float(__byte_perm(w, 0x3f000000u, 0x7044u | (k + 1) << 8)));
}

// Byte offset of the record of slab `slab` at slot (page, row).
__device__ __forceinline__ size_t record(int page, int row, int slab, int nslab, int page_size, int W)
{
    return (((size_t)page * nslab + slab) * page_size + row) * (size_t)(W * 5 / 4);
}

struct Write {
    const void *k, *v;
    int64_t ld;
    const int32_t *slots;
    int n, D, W, page_size, n_pages, shift;  // page_size = 1 << shift
    uint32_t page_bytes;
    uint8_t *pages;
    void *vk, *vv;
    int64_t ldv;
    int *status;
};

constexpr int kWriteWarps = 4;

// A lane per 8 channels of a row (k and v), `span` lanes a row: a warp takes
// 256 channels of a row (blockIdx.y which of them), or 32/span rows of fewer.
// Rows with a negative slot are left out.  Bound by HBM and issue alike: 65521
// rows of 2048 bf16 channels with their values back, 1.24 GB, take 264 us
// (0.73 of the measured copy rate), about 25 instructions a value, part of them
// for borders, which bf16 values meet often; with a division for the step and
// one a value it took 702 us.
template <typename T>
__global__ void __launch_bounds__(32 * kWriteWarps, 9) write_kernel(const __grid_constant__ Write p, int span)
{
    grid_dep_wait();  // programmatic dependent launch: inputs are ready
    grid_dep_launch();
    const int lane = threadIdx.x & 31, rows = 32 / span;
    const int ch = blockIdx.y * 256 + lane % span * 8;
    const int at = ch & (p.W - 1), rec_bytes = p.W / 4 * 5;
    uint8_t *base = p.pages + (size_t)(ch / p.W) * p.page_size * rec_bytes;
    const int step = gridDim.x * kWriteWarps * rows;
    // the warp's rows are the same number of rounds away for all its lanes
    for (int first = (blockIdx.x * kWriteWarps + (threadIdx.x >> 5)) * rows; first < p.n; first += step) {
        const int row = first + lane / span;
        const int slot = row < p.n && ch < p.D ? p.slots[row] : -1;
        const bool ok = slot >= 0 && slot < (int64_t)p.n_pages * p.page_size;
        float k[8] = {}, v[8] = {}, kc[8], vc[8];
        if (ok) {
            load8(static_cast<const T *>(p.k) + row * p.ld + ch, k);
            load8(static_cast<const T *>(p.v) + row * p.ld + ch, v);
        } else if (slot >= 0 && ch == 0) {
            atomicOr(p.status, DC_DEVERR_PAGE);
        }
        float ks, kl, vs, vl;
        const uint32_t kb = quantise8(k, ks, kl, kc), vb = quantise8(v, vs, vl, vc);
        if (step > INT32_MAX - first) first = INT32_MAX - step;  // the last round
        if (!ok) continue;
        uint8_t *rec = base + (size_t)(slot >> p.shift) * p.page_bytes + (slot & (p.page_size - 1)) * rec_bytes;
        *reinterpret_cast<uint2 *>(rec + at) = make_uint2(kb, vb);
        if (at % 32 == 0)
            *reinterpret_cast<uint2 *>(rec + p.W + at / 4) = make_uint2(pack_params(ks, kl), pack_params(vs, vl));
        if (p.vk) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                k[j] = fmaf(ks, kc[j], kl);
                v[j] = fmaf(vs, vc[j], vl);
            }
            store8(static_cast<T *>(p.vk) + row * p.ldv + ch, k);
            store8(static_cast<T *>(p.vv) + row * p.ldv + ch, v);
        }
    }
}

struct Decode {
    const void *qkv;  // [B, 3*D] rows: q | k | v
    int64_t ldq;
    const float *w;  // bias of head h: w + h * wh, row t at t * ldw
    int64_t ldw, wh;
    uint8_t *pages;
    const int32_t *table;
    int64_t ldtab;
    const int32_t *pos;
    int B, D, hs, W, nslab, n_pages, page_size, cap;
    float per_hs;  // 1 / hs
    uint32_t page_bytes;
    int shift;  // page_size = 1 << shift
    int w4;  // w's rows start on 16-byte boundaries
    void *Z;
    int64_t ldz;
    int *status;
    float *part;   // [gridDim.x][2][3][W]
    int *counter;  // [B * nslab], zero between launches
};

__device__ __forceinline__ float sigm(float q) { return 1.0f / (1.0f + __expf(-q)); }

__device__ __forceinline__ float ex2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Larger of two, NaN if either is: a NaN in the history reaches Z.
__device__ __forceinline__ float fmax_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr int kWarps = 4, kThreads = 32 * kWarps, kResident = 3;
constexpr int kRows = 16;  // history rows of a block: two halves, each within a page
constexpr int kStages = 2;  // blocks in flight of a warp
constexpr float kHuge = 0x1p24f;  // exponents of this size have no fraction in fp32
// (low - 16 step)^2 + step^2 of a row with a key of 2^23 or more is above this;
// a lane's sum of them may reach it from somewhat smaller keys on.  Summed
// packed (a maximum a row instead: 113.0 instead of 110.3 us at 32 x <=8191).
constexpr float kFar = 0x1p36f;
constexpr float kAbsorbs = 1e30f;  // beside a finite bias of this size keys below 2^23 vanish, in 64 bits too
// What an item costs a CTA besides its blocks, in blocks of 256 channels: this
// and the shares' other constants were measured at that slab width.
constexpr int kItem = 10;

// 16 bytes, of which the first `bytes` (0 or 16) are read, the others zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Blocks of kRows rows that position t's history has; 0: inactive.
__device__ __forceinline__ int row_blocks(const Decode &p, int t)
{
    return t < 0 || t >= p.cap ? 0 : t / kRows + 1;
}

__device__ __forceinline__ void join(float &m, float &num, float &den, float m2, float num2, float den2)
{
    const float mx = fmax_nan(m, m2), base = mx == -INFINITY ? 0.f : mx;  // masked so far: 0, or NaN of a value
    const float a = ex2(m - base), c = ex2(m2 - base);
    num = num * a + num2 * c;
    den = den * a + den2 * c;
    m = mx;
}

// One item again with a running maximum per channel, exponents and sums in 64
// bits, which no value, bias or number of positions overflows, by the whole
// CTA from the stored history (position t appended).  out holds (6 * kWarps +
// 1) * W floats; returns the W weighted means that it leaves there (0 where
// the bias masks every position).
template <int W>
__device__ __noinline__ const float *resum(const Decode &p, int b, int slab, int t, float *out)
{
    constexpr int LPR = W / 8, RPW = 32 / LPR;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LPR, oct = lane % LPR;
    const int ch = slab * W + oct * 8;
    const int32_t *tab = p.table + b * p.ldtab;
    const float *w = p.w + (ch / p.hs) * p.wh + t * p.ldw;
    double m[8], num[8], den[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        m[j] = -INFINITY;
        num[j] = den[j] = 0.;
    }
    auto add = [](double &m, double &num, double &den, double m2, double num2, double den2) {
        const double mx = m2 > m || m2 != m2 ? m2 : m;  // NaN if either is
        const double base = mx == -INFINITY ? 0. : mx;  // masked so far: 0, or NaN of a value
        const float a = ex2((float)((m - base) * 1.4426950408889634)), c = ex2((float)((m2 - base) * 1.4426950408889634));
        num = num * a + num2 * c;
        den = den * a + den2 * c;
        m = mx;
    };
    for (int i = warp * RPW + sub; i <= t; i += kWarps * RPW) {
        const int page = tab[i >> p.shift];
        if (page < 0 || page >= p.n_pages) continue;
        const uint8_t *rec = p.pages + record(page, i & (p.page_size - 1), slab, p.nslab, p.page_size, W);
        const uint2 code = *reinterpret_cast<const uint2 *>(rec + oct * 8);
        const uint2 par = *reinterpret_cast<const uint2 *>(rec + W + oct / 4 * 8);
        const double wi = w[i];
        double k[8], v[8];
        values8(code.x, par.x, k);
        values8(code.y, par.y, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) add(m[j], num[j], den[j], k[j] + wi, v[j], 1.);
    }
#pragma unroll
    for (int o = LPR; o < 32; o *= 2)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double m2 = __shfl_xor_sync(0xffffffffu, m[j], o), n2 = __shfl_xor_sync(0xffffffffu, num[j], o);
            add(m[j], num[j], den[j], m2, n2, __shfl_xor_sync(0xffffffffu, den[j], o));
        }
    // [kWarps][W] numerators, denominators, maxima; then the means [W]
    double *nums = reinterpret_cast<double *>(out), *dens = nums + kWarps * W, *tops = dens + kWarps * W;
    float *mean = reinterpret_cast<float *>(tops + kWarps * W);
    __syncthreads();
    if (sub == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            nums[warp * W + oct * 8 + j] = num[j];
            dens[warp * W + oct * 8 + j] = den[j];
            tops[warp * W + oct * 8 + j] = m[j];
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < W; c += kThreads) {
        double mc = tops[c], nc = nums[c], dc = dens[c];
        for (int g = 1; g < kWarps; ++g) add(mc, nc, dc, tops[g * W + c], nums[g * W + c], dens[g * W + c]);
        mean[c] = dc == 0. ? 0.f : (float)(nc / dc);
    }
    __syncthreads();
    return mean;
}

// The history of a slab (W channels of one sequence) is read once, in blocks
// of kRows rows, through a ring of blocks in flight that every warp keeps in
// shared memory.  A lane sums four rows of a block over one group of 32
// channels, so that the group's parameters and the bias are unpacked once for
// 32 channels: exponents y = log2(e) (k + w) in base 2, num, den = sums of
// 2^(y - ref) v and 2^(y - ref) in fp32, and one ref for the channels that
// share a bias (NH = 1: the group, else each 8), raised when a bound on y
// (the group's largest value is low + 15 step) passes it by more than 16.
//
// A channel that lies so far below its group that its den is below 2^-64 may
// have lost terms to underflow (a scale below 2^-126 becomes 0, and what it
// scales is at most 2^16 a position), and values may be so large (up to 1e37
// times a weight of up to 2^16) that num overflows, which leaves it infinite or
// NaN beside a finite den, or so small (below 2^-28) that num lies below 2^-90
// and may have lost terms too: such an item is then summed again, in 64 bits and
// with a running maximum per channel.  So are those whose exponents fp32 does
// not hold: references from 2^24 on (a row masked throughout by -1e9) and keys
// from 2^23 on, which a bias of their size may cancel.  Beside smaller keys a
// finite bias from 1e30 on (a mask of the type's lowest value) is the whole of
// the sum in 64 bits too, and the keys are left out.
//
// Work split: the row blocks of all (sequence, slab) items, one after the
// other, are cut into equal shares of q blocks, one share a CTA, so ragged
// lengths balance and a long sequence spreads over many CTAs; or, where that
// costs little, each item into parts of its own, so that a CTA has one.  An
// item that several CTAs share is merged, in CTA order, by the last of them
// to finish.
//
// What bounds it: a channel of a position costs one 2^x (8 cycles a warp and
// scheduler) and about 7 other instructions that overlap with it imperfectly
// (9.5 cycles alone), against 1.25 bytes of HBM, so 32 sequences of up to 8191
// positions, d = 2048 (345 MB, 53 us of HBM, 59 us of 2^x) take 110 us; the
// rest is what an item costs besides (merging, its first loads).  At 64
// sequences of 256-511 positions, d = 512, these are most of the 14.3 us.  Steps
// there: a lane per 8 channels 146 us (10.5 instructions a channel for
// unpacking and bounds), 16 channels 183 us (too few registers), a group of 32
// by four rows 141 us; codes through mixed-precision bf16 FMAs instead of byte
// permutations were as fast, four CTAs an SM (128 registers) 20% slower.
template <typename T, int W, int NH>
__global__ void __launch_bounds__(kThreads, kResident) decode_kernel(const __grid_constant__ Decode p)
{
    grid_dep_wait();  // programmatic dependent launch: inputs are ready
    grid_dep_launch();
    constexpr int LPR = W / 8;      // lanes of a block
    constexpr int RPW = 32 / LPR;   // blocks a warp reads at once
    constexpr int NG = W / 32;      // groups
    constexpr int kRec = W * 5 / 4, kStageBytes = RPW * kRows * kRec;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int sub = lane / LPR, oct = lane % LPR;
    const int group = lane % NG, rq = lane % LPR / NG * 4;  // this lane's group, first of its four rows
    // octets 2, 3 before 0, 1 in the upper four of 8 groups: no bank conflicts
    const int flip = W == 256 ? group >> 2 : 0;
    // each warp's blocks in flight; its partial sums [3][W] at the end
    extern __shared__ __align__(16) uint8_t ring_raw[];
    auto ring = reinterpret_cast<uint8_t(*)[kStages][kStageBytes]>(ring_raw);
    auto part = [&](int warp) { return reinterpret_cast<float *>(ring[warp][0]); };
    static_assert(kStages * kStageBytes >= 8 * 1024, "room for the lanes' sums");
    static_assert(kWarps * kStages * kStageBytes >= (6 * kWarps + 1) * W * 4, "room for resum's");
    const uint32_t mine = smem_u32(ring[warp][0]) + sub * (kRows * kRec) + oct * 16;
    __shared__ int s_sum[kWarps], s_max[kWarps], s_active[kWarps], s_b, s_first, s_t, s_last;

    int sum = 0, most = 0, active = 0, t = -1, nb = 0, inc = 0;
    for (int b = tid; b < p.B; b += kThreads) {
        t = p.pos[b];
        nb = row_blocks(p, t);
        sum += nb;
        most = max(most, nb);
        active += nb > 0;
        if (nb == 0 && b % gridDim.x == blockIdx.x) {  // an inactive sequence
            if (t >= 0) atomicOr(p.status, DC_DEVERR_FULL);
            const float zero[8] = {};
            for (int c = 0; c < p.D; c += 8) store8(static_cast<T *>(p.Z) + b * p.ldz + c, zero);
        }
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    most = __reduce_max_sync(0xffffffffu, most);
    active = __reduce_add_sync(0xffffffffu, active);
    if (lane == 0) {
        s_sum[warp] = sum;
        s_max[warp] = most;
        s_active[warp] = active;
    }
    if (tid == 0) s_b = -1;
    __syncthreads();
    sum = most = active = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
        sum += s_sum[k];
        most = max(most, s_max[k]);
        active += s_active[k];
    }
    // the plan fits 32 bits (the entry point sees to it): divisions of 64 took
    // 1 us of a call
    const int total = sum * p.nslab, items = active * p.nslab;
    if (items == 0) return;
    const int units = total + items * kItem, G = gridDim.x;
    // at least some rounds of the CTA's warps, so that merging a long sequence's
    // shares does not outweigh summing them (1 x 8192 positions, d = 1024: 18.2
    // us; half as many rounds 21.1)
    const int least = min(most, kWarps * ((int)sqrtf((float)most) / 16 + 1));
    int q = max((units + G - 1) / G, least);
    // even: every item in ceil(nb / q) equal parts of its own, one a CTA, where
    // that makes no CTA's share much longer (128 sequences of up to 1024
    // positions, d = 256: 17.6 us, without 19.0)
    const int even_q = 2 * items <= G ? max((total + G - items - 1) / (G - items), least) : INT32_MAX;
    const bool even = even_q <= q + 6;
    if (even) q = even_q;
    const int fewer = (q - 1) / (kWarps * RPW) * (kWarps * RPW);
    if (even && p.B <= kThreads && fewer >= max(1, least)) {
        // parts of one round of the warps less, where rounding leaves the CTAs
        // (64 sequences of 256-511 positions, d = 512: 15.9 -> 15.2 us)
        const int parts = __reduce_add_sync(0xffffffffu, (nb + fewer - 1) / fewer);
        __syncthreads();
        if (lane == 0) s_sum[warp] = parts;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) all += s_sum[k];
        if (all * p.nslab <= G) q = fewer;
    }
    auto weight = [&](int nb) {  // CTAs, or blocks and what an item costs besides
        return nb == 0 ? 0 : even ? (nb + q - 1) / q : nb + kItem;
    };
    // this CTA's share: [u, u1) of all slabs' weights, one sequence after the other
    int u = even ? blockIdx.x : blockIdx.x * q;
    int u1 = even ? u + 1 : min(units, u + q);
    // the sequence that u lies in: the weight before it
    const int target = u / p.nslab;
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += kThreads) {
        if (p.B > kThreads) {
            t = b0 + tid < p.B ? p.pos[b0 + tid] : -1;
            nb = row_blocks(p, t);
        }
        const int own = weight(nb);
        inc = own;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        __syncthreads();
        if (lane == 31) s_sum[warp] = inc;
        __syncthreads();
        int at = before + inc - own;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            if (k < warp) at += s_sum[k];
            before += s_sum[k];
        }
        if (target >= at && target < at + own) {
            s_b = b0 + tid;
            s_first = at;
            s_t = t;
        }
        __syncthreads();
        if (s_b >= 0) break;
    }
    int b = s_b;
    if (b < 0) return;  // behind the last share
    t = s_t;
    nb = row_blocks(p, t);
    const int local = u - s_first * p.nslab, own = weight(nb);
    int slab = local / own, off = local % own;  // off: units of the item before the share
    int j0 = blockIdx.x - off, j1 = j0 + own - 1;
    if (even) {  // part off of own: its blocks, as units behind the item's kItem
        u1 = kItem + (uint32_t)((off + 1) * nb) / (uint32_t)own;
        off = kItem + (uint32_t)(off * nb) / (uint32_t)own;
        u = off;
    }

    for (;;) {
        const int taken = min(nb + kItem - off, u1 - u);
        const int blk = max(0, off - kItem), n = off + taken - kItem - blk;  // the share's blocks
        const int u_item = u - off;
        if (n > 0) {
            const int32_t *tab = p.table + b * p.ldtab;
            const T *row = static_cast<const T *>(p.qkv) + b * p.ldq + slab * W;
            // exact below 2^21
            auto head_of = [&](int channel) { return (int)((channel + 0.5f) * p.per_hs); };
            const float *w[NH];  // bias rows of this lane's octets
#pragma unroll
            for (int h = 0; h < NH; ++h)
                w[h] = p.w + head_of(slab * W + group * 32 + (h ^ (2 * flip)) * 8 * (NH > 1)) * p.wh + t * p.ldw + rq;
            // this warp's blocks: k0, k0 + step, ... < n, RPW neighbours at once
            constexpr int kStep = kWarps * RPW;
            const int k0 = warp * RPW + sub;
            const int rounds = max(0, (n - warp * RPW + kStep - 1) / kStep);
            uint8_t *pool = p.pages + (size_t)slab * p.page_size * kRec;
            // pages of a block's halves, -1 behind t and past the share
            auto pages_of = [&](int it) {
                const int k = k0 + it * kStep, i0 = (blk + k) * kRows;
                return make_int2(k < n ? tab[i0 >> p.shift] : -1, k < n && i0 + 8 <= t ? tab[(i0 + 8) >> p.shift] : -1);
            };
            auto there = [&](int page) { return (uint32_t)page < (uint32_t)p.n_pages; };
            auto record_of = [&](int i, int page) {
                return pool + (size_t)(uint32_t)page * p.page_bytes + (uint32_t)(i & (p.page_size - 1)) * kRec;
            };
            // a half without a page is filled with zeros
            auto fetch = [&](int it, int2 page) {
                const int i0 = (blk + k0 + it * kStep) * kRows;
                const uint32_t dst = mine + (it % kStages) * kStageBytes;
                const bool a = there(page.x), c = there(page.y);
                const uint8_t *s0 = record_of(i0, a ? page.x : 0) + oct * 16;
                const uint8_t *s1 = record_of(i0 + 8, c ? page.y : 0) + oct * 16;
#pragma unroll
                for (int k = 0; k < 5; ++k) cp_async16(dst + k * (LPR * 16), s0 + k * (LPR * 16), a ? 16 : 0);
#pragma unroll
                for (int k = 0; k < 5; ++k) cp_async16(dst + (5 + k) * (LPR * 16), s1 + k * (LPR * 16), c ? 16 : 0);
                cp_async_commit();
            };
            // biases of this lane's rows, -inf behind t and without a page
            auto biases = [&](int it, int2 page, float4 (&x)[NH]) {
                const int i0 = (blk + k0 + it * kStep) * kRows;
                const int left = there(rq < 8 ? page.x : page.y) ? t - i0 - rq : -1;
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const float *src = w[h] + i0;
                    if (p.w4 && left >= 3)
                        x[h] = *reinterpret_cast<const float4 *>(src);
                    else
                        x[h] = make_float4(left >= 0 ? src[0] : -INFINITY, left >= 1 ? src[1] : -INFINITY,
                                           left >= 2 ? src[2] : -INFINITY, left >= 3 ? src[3] : -INFINITY);
                }
            };
            // position t: the lanes of its block quantise it, 8 channels each
            const int tail = nb - 1 - blk - k0;  // rounds * kStep on, if it is this warp's
            const bool owner = tail >= 0 && tail % kStep == 0 && nb - 1 - blk < n;
            float fresh[2][8];
            int home = -1;
            if (owner) {
                load8(row + p.D + oct * 8, fresh[0]);
                load8(row + 2 * p.D + oct * 8, fresh[1]);
                home = tab[t >> p.shift];
            }
            // pages of the blocks in flight, the next one's at hand early
            int2 page[kStages];
#pragma unroll
            for (int s = 0; s < kStages; ++s) page[s] = pages_of(s);
#pragma unroll
            for (int s = 0; s < kStages - 1; ++s) fetch(s, page[s]);
            float4 wn[NH];
            biases(0, page[0], wn);
            uint2 nc = make_uint2(0, 0), np = nc;  // its codes and parameters
            if (owner && there(home)) {
                float st, lo, c[8];
                const uint32_t lanes = 0xfu << (lane & ~3);
                nc.x = quantise8(fresh[0], st, lo, c, lanes);
                np.x = pack_params(st, lo);
                nc.y = quantise8(fresh[1], st, lo, c, lanes);
                np.y = pack_params(st, lo);
                uint8_t *rec = record_of(t, home);
                *reinterpret_cast<uint2 *>(rec + oct * 8) = nc;
                if (oct % 4 == 0) *reinterpret_cast<uint2 *>(rec + W + oct * 2) = np;
            }

            // octet o, pair j (factors)
            f32x2 num[4][4], den[4][4];
            float ref[NH];
            f32x2 far = 0;  // sums of the keys' (low - 16 step)^2 and step^2
#pragma unroll
            for (int o = 0; o < 4; ++o)
#pragma unroll
                for (int j = 0; j < 4; ++j) num[o][j] = den[o][j] = 0;
#pragma unroll
            for (int h = 0; h < NH; ++h) ref[h] = -INFINITY;
#pragma unroll 1
            for (int it = 0; it < rounds; ++it) {
                fetch(it + kStages - 1, page[kStages - 1]);
                const int2 now = page[0];
#pragma unroll
                for (int s = 0; s < kStages - 1; ++s) page[s] = page[s + 1];
                page[kStages - 1] = pages_of(it + kStages);
                float4 wl[NH];
#pragma unroll
                for (int h = 0; h < NH; ++h) wl[h] = wn[h];
                biases(it + 1, page[0], wn);
                cp_async_wait<kStages - 1>();
                __syncwarp();
                uint8_t *stage = ring[warp][it % kStages] + sub * (kRows * kRec);
                const int at = k0 + it * kStep < n ? t - (blk + k0 + it * kStep) * kRows : -1;
                if (__any_sync(0xffffffffu, at < kRows || !there(now.x) || !there(now.y))) {
                    // position t itself, or a half without a page
                    if (at >= 0 && oct == 0 && (!there(now.x) || (at >= 8 && !there(now.y))))
                        atomicOr(p.status, DC_DEVERR_PAGE);
                    if (at >= 0 && at < kRows) {  // and nothing behind it
                        for (int r = at; r < kRows; ++r) {
                            uint8_t *to = stage + r * kRec;
                            *reinterpret_cast<uint2 *>(to + oct * 8) = r > at ? make_uint2(0, 0) : nc;
                            if (oct % 4 == 0)
                                *reinterpret_cast<uint2 *>(to + W + oct * 2) = r > at ? make_uint2(0, 0) : np;
                        }
                    }
                    __syncwarp();
                }
                // one test for the four rows (112.1 -> 109.5 us at 32 x <=8191
                // positions; with four biases a row one each is as fast)
                bool odd = false;
#pragma unroll
                for (int h = 0; h < NH; ++h)
                    odd |= fmaxf(fmaxf(fabsf(wl[h].x), fabsf(wl[h].y)), fmaxf(fabsf(wl[h].z), fabsf(wl[h].w))) >= kAbsorbs;
                // rows whose exponents are bounded together: fewer branches between
                // the sums (two with one bias a row: 116.6 -> 113 us; else one, for registers)
                constexpr int kTogether = NH == 1 ? 2 : 1;
#pragma unroll
                for (int r0 = 0; r0 < 4; r0 += kTogether) {
                    // y - ref = ka + ks (1/2 + c/32), v = va + vs (1/2 + c/32):
                    // value = low + step c = (low - 16 step) + 32 step (1/2 + c/32),
                    // exact in fp32 unless low outweighs step 2^15 times
                    float ks[kTogether][NH], ka[kTogether][NH], vs[kTogether], va[kTogether], top[NH];
#pragma unroll
                    for (int h = 0; h < NH; ++h) top[h] = -INFINITY;
#pragma unroll
                    for (int i = 0; i < kTogether; ++i) {
                        const int r = r0 + i;
                        const uint2 par = *reinterpret_cast<const uint2 *>(stage + (rq + r) * kRec + W + group * 8);
                        const float kstep = __uint_as_float(par.x << 16), vstep = __uint_as_float(par.y << 16);
                        const float klow = fmaf(kstep, -16.f, __uint_as_float(par.x & 0xffff0000u));
                        va[i] = fmaf(vstep, -16.f, __uint_as_float(par.y & 0xffff0000u));
                        vs[i] = 32.f * vstep;
                        far = fma2(pack2(klow, kstep), pack2(klow, kstep), far);
#pragma unroll
                        for (int h = 0; h < NH; ++h) {
                            const float x = r == 0 ? wl[h].x : r == 1 ? wl[h].y : r == 2 ? wl[h].z : wl[h].w;
                            ks[i][h] = kstep * (32.f * kLog2e);
                            ka[i][h] = (klow + x) * kLog2e;
                            if ((NH > 1 || odd) && fabsf(x) >= kAbsorbs && x > -INFINITY) {
                                // any factor serves that keeps it finite
                                ks[i][h] = 0.f;
                                ka[i][h] = 0.5f * x;
                            }
                            top[h] = fmax_nan(top[h], fmaf(ks[i][h], 31.f / 32.f, ka[i][h]));
                        }
                    }
#pragma unroll
                    for (int h = 0; h < NH; ++h) {
                        if (!(top[h] <= ref[h] + 16.f)) {  // also where either is NaN
                            const float scale = ex2(ref[h] - top[h]);
#pragma unroll
                            for (int o = 0; o < 4; ++o)
                                if (NH == 1 || o == h)
#pragma unroll
                                    for (int j = 0; j < 4; ++j) {
                                        num[o][j] = mul2(num[o][j], pack2(scale, scale));
                                        den[o][j] = mul2(den[o][j], pack2(scale, scale));
                                    }
                            ref[h] = top[h];
                        }
                        const float base = ref[h] == -INFINITY ? 0.f : ref[h];
#pragma unroll
                        for (int i = 0; i < kTogether; ++i) ka[i][h] -= base;
                    }
#pragma unroll
                    for (int i = 0; i < kTogether; ++i) {
                        const uint8_t *rec = stage + (rq + r0 + i) * kRec;
                        uint2 code[4];
                        if (kRec % 16 == 0) {
                            const uint4 c = *reinterpret_cast<const uint4 *>(rec + group * 32 + 16 * flip);
                            const uint4 d = *reinterpret_cast<const uint4 *>(rec + group * 32 + 16 - 16 * flip);
                            code[0] = make_uint2(c.x, c.y);
                            code[1] = make_uint2(c.z, c.w);
                            code[2] = make_uint2(d.x, d.y);
                            code[3] = make_uint2(d.z, d.w);
                        } else {
#pragma unroll
                            for (int o = 0; o < 4; ++o)
                                code[o] = *reinterpret_cast<const uint2 *>(rec + group * 32 + (o ^ (2 * flip)) * 8);
                        }
                        f32x2 ks2[NH], ka2[NH];
                        const f32x2 vs2 = pack2(vs[i], vs[i]), va2 = pack2(va[i], va[i]);
#pragma unroll
                        for (int h = 0; h < NH; ++h) {
                            ks2[h] = pack2(ks[i][h], ks[i][h]);
                            ka2[h] = pack2(ka[i][h], ka[i][h]);
                        }
#pragma unroll
                        for (int o = 0; o < 4; ++o) {
                            const int h = NH == 1 ? 0 : o;
                            const uint32_t k0 = code[o].x << 3 & 0x78787878u, k1 = code[o].x >> 1 & 0x78787878u;
                            const uint32_t v0 = code[o].y << 3 & 0x78787878u, v1 = code[o].y >> 1 & 0x78787878u;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float2 y = unpack2(fma2(factors(k0, k1, j), ks2[h], ka2[h]));
                                const f32x2 e = pack2(ex2(y.x), ex2(y.y));
                                const f32x2 v = fma2(factors(v0, v1, j), vs2, va2);
                                num[o][j] = fma2(e, v, num[o][j]);
                                den[o][j] = add2(den[o][j], e);
                            }
                        }
                    }
                }
                __syncwarp();  // the stage may be filled again
            }
            cp_async_wait<0>();
            __syncwarp();
            constexpr int CPT = (W + kThreads - 1) / kThreads;  // channels a thread finishes
            float qv[CPT];  // at hand for the end (15.2 -> 15.0 us at 64 x 256-511 positions)
#pragma unroll
            for (int k = 0; k < CPT; ++k) qv[k] = to_f<T>(row[min(tid + k * kThreads, W - 1)]);
            // the lanes of a group: one ref, then sums over their NL lanes
            constexpr int NL = 32 / NG;
            float *sums = part(warp);  // [NL][2][W], then ref, num, den [3][W]
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                const float keys = unpack2(far).x + unpack2(far).y;
                if (!(keys < kFar)) ref[h] = keys * INFINITY;  // or NaN, which reaches Z
                float r = ref[h];
#pragma unroll
                for (int x = NG; x < 32; x *= 2) r = fmax_nan(r, __shfl_xor_sync(0xffffffffu, r, x));
                const float scale = ref[h] == -INFINITY ? 0.f : ex2(ref[h] - r);
                ref[h] = r;
#pragma unroll
                for (int o = 0; o < 4; ++o)
                    if (NH == 1 || o == h)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            num[o][j] = mul2(num[o][j], pack2(scale, scale));
                            den[o][j] = mul2(den[o][j], pack2(scale, scale));
                        }
            }
#pragma unroll
            for (int o = 0; o < 4; ++o) {
                float *to = sums + (lane / NG) * 2 * W + group * 32 + (o ^ (2 * flip)) * 8;
                float2 m[4], d[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m[j] = unpack2(num[o][j]);
                    d[j] = unpack2(den[o][j]);
                }
                store8(to, {m[0].x, m[2].x, m[0].y, m[2].y, m[1].x, m[3].x, m[1].y, m[3].y});
                store8(to + W, {d[0].x, d[2].x, d[0].y, d[2].y, d[1].x, d[3].x, d[1].y, d[3].y});
            }
            __syncwarp();
            float sn[W / 32], sd[W / 32];
#pragma unroll
            for (int k = 0; k < W / 32; ++k) {
                sn[k] = sd[k] = 0.f;
#pragma unroll (NL < 8 ? NL : 8)
                for (int l = 0; l < NL; ++l) {
                    sn[k] += sums[l * 2 * W + k * 32 + lane];
                    sd[k] += sums[(l * 2 + 1) * W + k * 32 + lane];
                }
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < W / 32; ++k) {
                sums[W + k * 32 + lane] = sn[k];
                sums[2 * W + k * 32 + lane] = sd[k];
            }
#pragma unroll
            for (int o = 0; o < 4; ++o)
                if (lane / NG == o) {
                    const float r = ref[o % NH];
                    store8(sums + group * 32 + (o ^ (2 * flip)) * 8, {r, r, r, r, r, r, r, r});
                }
            __syncthreads();
            float fm[CPT], fn[CPT], fd[CPT];
#pragma unroll
            for (int k = 0; k < CPT; ++k) {
                const int c = tid + k * kThreads;
                if (c >= W) continue;
                fm[k] = part(0)[c];
                fn[k] = part(0)[W + c];
                fd[k] = part(0)[2 * W + c];
#pragma unroll
                for (int g = 1; g < kWarps; ++g)
                    join(fm[k], fn[k], fd[k], part(g)[c], part(g)[W + c], part(g)[2 * W + c]);
            }
            bool finish = n == nb;
            if (!finish) {  // shared with other CTAs
                // second slot: an item that begins inside the CTA's share
                const auto slot = [&](int g) { return (int64_t)g * 2 + (!even && u_item > g * q); };
                float *mine = p.part + slot(blockIdx.x) * 3 * W;
#pragma unroll
                for (int k = 0; k < CPT; ++k) {
                    const int c = tid + k * kThreads;
                    if (c >= W) continue;
                    mine[c] = fm[k];
                    mine[W + c] = fn[k];
                    mine[2 * W + c] = fd[k];
                }
                __threadfence();
                __syncthreads();
                if (!even) {
                    j0 = (u_item + kItem) / q;
                    j1 = (u_item + kItem + nb - 1) / q;
                }
                if (tid == 0) {
                    int *counter = p.counter + (int64_t)b * p.nslab + slab;
                    s_last = atomicAdd(counter, 1) == j1 - j0;
                    if (s_last) *counter = 0;  // ready for the next launch
                }
                __syncthreads();
                if (s_last) {
                    finish = true;
                    __threadfence();
#pragma unroll
                    for (int k = 0; k < CPT; ++k) {
                        fm[k] = -INFINITY;
                        fn[k] = fd[k] = 0.f;
                    }
                    int g0 = j0;
                    // the next N shares, whose sums are read at once (8 at a time: 1 x
                    // 8192 positions, d = 1024, 21.0 us instead of 18.6)
                    const auto merge = [&](auto count) {
                        constexpr int N = decltype(count)::value;
                        float x[N][CPT][3];
#pragma unroll
                        for (int d = 0; d < N; ++d) {
                            const float *src = p.part + slot(min(g0 + d, j1)) * 3 * W;
#pragma unroll
                            for (int k = 0; k < CPT; ++k) {
                                const int c = min(tid + k * kThreads, W - 1);
                                x[d][k][0] = __ldcg(src + c);
                                x[d][k][1] = __ldcg(src + W + c);
                                x[d][k][2] = __ldcg(src + 2 * W + c);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < CPT; ++k) {
                            float top = fm[k];
#pragma unroll
                            for (int d = 0; d < N; ++d) top = fmax_nan(top, x[d][k][0]);
                            const float base = top == -INFINITY ? 0.f : top;  // masked so far: 0, or NaN of a value
                            const float a = ex2(fm[k] - base);
                            fn[k] *= a;
                            fd[k] *= a;
                            fm[k] = top;
#pragma unroll
                            for (int d = 0; d < N; ++d) {
                                if (g0 + d > j1) continue;
                                const float c = ex2(x[d][k][0] - base);
                                fn[k] = fmaf(x[d][k][1], c, fn[k]);
                                fd[k] = fmaf(x[d][k][2], c, fd[k]);
                            }
                        }
                        g0 += N;
                    };
                    while (g0 + 8 <= j1) merge(std::integral_constant<int, 16>{});
                    if (g0 + 4 <= j1) merge(std::integral_constant<int, 8>{});
                    else if (g0 <= j1) merge(std::integral_constant<int, 4>{});
                }
            }
            if (finish) {
                bool lost = false;
#pragma unroll
                for (int k = 0; k < CPT; ++k) {
                    if (tid + k * kThreads >= W || fm[k] == -INFINITY) continue;
                    const float far = fabsf(fm[k]);
                    lost |= (far >= kHuge && far < 0.5f * kAbsorbs) || far == INFINITY || fd[k] < 0x1p-64f ||
                            (fd[k] < INFINITY && !(fabsf(fn[k]) < INFINITY)) ||
                            (fabsf(fn[k]) < 0x1p-90f && (fn[k] != 0.f || fd[k] < 0x1p-32f));
                }
                if (__syncthreads_or(lost)) {
                    const float *mean = resum<W>(p, b, slab, t, part(0));
#pragma unroll
                    for (int k = 0; k < CPT; ++k) {
                        const int c = tid + k * kThreads;
                        if (c >= W) continue;
                        fn[k] = mean[c];
                        fd[k] = 1.f;
                    }
                }
#pragma unroll
                for (int k = 0; k < CPT; ++k) {
                    const int c = tid + k * kThreads;
                    if (c >= W) continue;
                    static_cast<T *>(p.Z)[b * p.ldz + slab * W + c] =
                        from_f<T>(fd[k] == 0.f ? 0.f : sigm(qv[k]) * (fn[k] / fd[k]));
                }
            }
        }
        u += taken;
        if (u >= u1) return;
        off = 0;
        if (++slab == p.nslab) {
            slab = 0;
            do {  // u < total: there is another active one
                if (++b >= p.B) return;
                t = p.pos[b];
            } while ((nb = row_blocks(p, t)) == 0);
        }
        __syncthreads();  // part is reused
    }
}

static int decode_grid() { return kResident * sm_count(); }

// Partial sums come first, in room for the widest slab, then the counters: a
// workspace serves calls of any smaller batch or width in between.
static size_t part_bytes() { return (size_t)decode_grid() * 2 * 3 * 256 * sizeof(float); }

template <typename T, int W>
static cudaError_t launch_slab(const Decode &p, cudaStream_t st)
{
    const dim3 grid((unsigned)decode_grid()), block(kThreads);
    constexpr int smem = kWarps * kStages * (256 / W) * kRows * (W * 5 / 4);
    // a bias for a group where heads allow it (32 sequences of up to 8191
    // positions, hs = 128: 110 us; hs = 120, d = 1920, a bias for each 8: 163)
    auto kernel = p.hs % 32 == 0 ? decode_kernel<T, W, 1> : decode_kernel<T, W, 4>;
    static SmemOnce once[2];
    const cudaError_t e = once[p.hs % 32 == 0].set(kernel, smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, grid, block, smem, st, 1, p);
}

template <typename T>
static cudaError_t launch_decode(const Decode &p, cudaStream_t st)
{
    switch (p.W) {
        case 256: return launch_slab<T, 256>(p, st);
        case 128: return launch_slab<T, 128>(p, st);
        case 64: return launch_slab<T, 64>(p, st);
        default: return launch_slab<T, 32>(p, st);
    }
}

static int check_pool(int D, int n_pages, int page_size)
{
    if (D <= 0 || D % 32 || D > 1 << 20)
        return fail(DC_ERR_INVALID, "D must be a positive multiple of 32, at most 2^20 (got %d)", D);
    if (n_pages <= 0) return fail(DC_ERR_INVALID, "n_pages must be positive");
    if (page_size < 8 || page_size > 256 || (page_size & (page_size - 1)))
        return fail(DC_ERR_INVALID, "page_size must be 8, 16, 32, 64, 128 or 256 (got %d)", page_size);
    if ((int64_t)n_pages * page_size > INT32_MAX)
        return fail(DC_ERR_INVALID, "n_pages * page_size must be below 2^31");
    return DC_OK;
}

}  // namespace kv4
}  // namespace dc

using namespace dc;

extern "C" {

int dc_kv4_pages_size(int n_pages, int page_size, int D, size_t *bytes)
{
    clear_error();
    DC_TRY(kv4::check_pool(D, n_pages, page_size));
    if (!bytes) return fail(DC_ERR_INVALID, "null pointer");
    *bytes = (size_t)n_pages * page_size * D / 4 * 5;
    return DC_OK;
}

int dc_kv4_write(const void *k, const void *v, int ld, int dtype, const int32_t *slots, int n, int D,
                 void *pages, int n_pages, int page_size, void *values_k, void *values_v, int ldv,
                 void *stream)
{
    using namespace dc::kv4;
    clear_error();
    DC_TRY(check_pool(D, n_pages, page_size));
    if (dtype != DC_F32 && dtype != DC_BF16) return fail(DC_ERR_INVALID, "bad dtype %d", dtype);
    if (n < 0 || n > INT32_MAX - 64) return fail(DC_ERR_INVALID, "bad row count %d", n);
    if (n == 0) return DC_OK;
    if (!k || !v || !slots || !pages) return fail(DC_ERR_INVALID, "null pointer");
    if (!values_k != !values_v) return fail(DC_ERR_INVALID, "values_k and values_v go together");
    const int per16 = dtype == DC_F32 ? 4 : 8;
    if (ld < D || ld % per16 || (values_k && (ldv < D || ldv % per16)))
        return fail(DC_ERR_INVALID, "row strides must be at least D and multiples of 16 bytes");
    if (!aligned16(k) || !aligned16(v) || !aligned16(pages) || !aligned16(values_k) || !aligned16(values_v))
        return fail(DC_ERR_INVALID, "k, v, pages and the values need 16-byte alignment");
    Write p{};
    p.k = k;
    p.v = v;
    p.ld = ld;
    p.slots = slots;
    p.n = n;
    p.D = D;
    p.W = slab_width(D);
    p.page_size = page_size;
    for (p.shift = 3; 1 << p.shift < page_size;) ++p.shift;
    p.page_bytes = (uint32_t)(page_size * (int64_t)D * 5 / 4);
    p.n_pages = n_pages;
    p.pages = static_cast<uint8_t *>(pages);
    p.vk = values_k;
    p.vv = values_v;
    p.ldv = ldv;
    p.status = device_status_word();
    if (!p.status) return fail(DC_ERR_CUDA, "no device status word");
    cudaStream_t st = as_stream(stream);
    KernelTimer kt("kv4_write", st);
    int span = 4;  // lanes a row
    while (span < 32 && span * 8 < D) span *= 2;
    const int chunks = (D + 255) / 256, rows = kWriteWarps * (32 / span);
    const int most = std::max(1, sm_count() * 64 / chunks);
    const dim3 grid(std::min((n - 1) / rows + 1, most), chunks), block(32 * kWriteWarps);
    DC_CUDA_TRY(dtype == DC_F32 ? launch_pdl(write_kernel<float>, grid, block, 0, st, 1, p, span)
                                : launch_pdl(write_kernel<__nv_bfloat16>, grid, block, 0, st, 1, p, span));
    return DC_OK;
}

size_t dc_aft_decode4_workspace_size(int B, int D)
{
    const int W = D > 0 ? kv4::slab_width(D) : 0;
    if (B <= 0 || !W) return 0;
    // counters for the narrowest slabs: the size grows with B and D
    return kv4::part_bytes() + round_up((int64_t)B * (D / 32) * sizeof(int), 256);
}

int dc_aft_decode4(const void *qkv, int ldq, int dtype, const float *w, int ldw, long long head_stride_w,
                   void *pages, int n_pages, int page_size, const int32_t *table, int ldtab, int B, int H,
                   int hs, const int32_t *pos, int Tmax, void *Z, int ldz, void *workspace,
                   size_t workspace_bytes, void *stream)
{
    using namespace dc::kv4;
    clear_error();
    if (B < 0 || H <= 0 || hs <= 0 || Tmax <= 0 || ldtab <= 0 || (int64_t)H * hs > INT32_MAX / 4)
        return fail(DC_ERR_INVALID, "bad decode shape B=%d H=%d hs=%d Tmax=%d ldtab=%d", B, H, hs, Tmax, ldtab);
    const int D = H * hs;
    DC_TRY(check_pool(D, n_pages, page_size));
    if (hs % 8) return fail(DC_ERR_INVALID, "hs must be a multiple of 8 (got %d)", hs);
    if (dtype != DC_F32 && dtype != DC_BF16) return fail(DC_ERR_INVALID, "bad dtype %d", dtype);
    if (B == 0) return DC_OK;
    const int per16 = dtype == DC_F32 ? 4 : 8;
    if (ldq < 3 * D || ldq % per16 || ldz < D || ldz % per16 || ldw < Tmax)
        return fail(DC_ERR_INVALID, "ldq >= 3D and ldz >= D must be multiples of 16 bytes, ldw >= Tmax");
    if (!qkv || !w || !pages || !table || !pos || !Z || !workspace) return fail(DC_ERR_INVALID, "null pointer");
    if (!aligned16(qkv) || !aligned16(pages) || !aligned16(Z) || !aligned16(workspace))
        return fail(DC_ERR_INVALID, "qkv, pages, Z and the workspace need 16-byte alignment");
    if (workspace_bytes < dc_aft_decode4_workspace_size(B, D))
        return fail(DC_ERR_NOMEM, "decode workspace too small");
    Decode p{};
    p.qkv = qkv;
    p.ldq = ldq;
    p.w = w;
    p.ldw = ldw;
    p.wh = head_stride_w;
    p.pages = static_cast<uint8_t *>(pages);
    p.table = table;
    p.ldtab = ldtab;
    p.pos = pos;
    p.B = B;
    p.D = D;
    p.hs = hs;
    p.per_hs = 1.f / hs;
    p.W = slab_width(D);
    p.nslab = D / p.W;
    p.n_pages = n_pages;
    p.page_size = page_size;
    p.cap = (int)std::min<int64_t>(Tmax, (int64_t)ldtab * page_size);
    for (p.shift = 3; 1 << p.shift < page_size;) ++p.shift;
    p.page_bytes = (uint32_t)(page_size * (int64_t)D * 5 / 4);
    p.w4 = aligned16(w) && ldw % 4 == 0 && head_stride_w % 4 == 0;
    p.part = static_cast<float *>(workspace);
    p.counter = reinterpret_cast<int *>(static_cast<char *>(workspace) + part_bytes());
    p.Z = Z;
    p.ldz = ldz;
    // the kernel's plan in 32 bits
    const int blocks = p.cap / kRows + 1;
    if (blocks > 65536 || (double)B * p.nslab * (blocks + kItem) > (1 << 30))
        return fail(DC_ERR_INVALID, "Tmax must be below 2^20, and B * D * Tmax is limited (B=%d D=%d Tmax=%d)", B, D, Tmax);
    p.status = device_status_word();
    if (!p.status) return fail(DC_ERR_CUDA, "no device status word");
    cudaStream_t st = as_stream(stream);
    KernelTimer kt("aft_decode4", st);
    DC_CUDA_TRY(dtype == DC_F32 ? launch_decode<float>(p, st) : launch_decode<__nv_bfloat16>(p, st));
    return DC_OK;
}

}  // extern "C"
