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
// <= step / 2.  A group with a value that is not finite (or above 1e38 in
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

#include "dc_internal.h"
#include "dc_ptx.cuh"

namespace dc {
namespace kv4 {

constexpr float kBig = 1e38f;        // larger magnitudes count as not finite
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

// One group's quantisation by the 4 lanes (xor 1, 2) that hold its 32 values:
// step and low (bf16 values, the same on the 4 lanes), this lane's 8 codes.
// `lanes`: the lanes that take part, whole groups.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], float &step, float &low,
                                              uint32_t lanes = 0xffffffffu)
{
    float mn = x[0], mx = x[0];
    int bad = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        mn = fminf(mn, x[j]);
        mx = fmaxf(mx, x[j]);
        bad |= !(fabsf(x[j]) <= kBig);
    }
#pragma unroll
    for (int o = 1; o <= 2; o *= 2) {
        mn = fminf(mn, __shfl_xor_sync(lanes, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(lanes, mx, o));
        bad |= __shfl_xor_sync(lanes, bad, o);
    }
    if (bad) {
        step = __uint_as_float(0x7fff0000u);
        low = 0.f;
        return 0;
    }
    uint32_t cut = __float_as_uint(mn) & 0xffff0000u;  // towards zero
    if (__uint_as_float(cut) > mn) cut += 0x10000u;
    low = __uint_as_float(cut == 0x80000000u ? 0u : cut);  // -0 is stored as 0
    const float up = __fdiv_ru(__fsub_ru(mx, low), 15.f);
    step = __uint_as_float((__float_as_uint(up) + 0xffffu) & 0xffff0000u);
    if (step == 0.f) {  // -0 - 0 among them
        step = 0.f;
        return 0;
    }
    uint32_t codes = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float c = fminf(fmaxf(floorf(__fdiv_rn(x[j] - low, step) + 0.5f), 0.f), 15.f);
        // the estimate is within one of the code; the borders decide
        if (c > 0.f && x[j] < __fmaf_ru(step, c - 0.5f, low))
            c -= 1.f;
        else if (c < 15.f && x[j] >= __fmaf_ru(step, c + 0.5f, low))
            c += 1.f;
        codes |= (uint32_t)c << (4 * j);
    }
    return codes;
}

__device__ __forceinline__ uint32_t pack_params(float step, float low)
{
    return (__float_as_uint(step) >> 16) | (__float_as_uint(low) & 0xffff0000u);
}

// The 8 values that codes stand for.
__device__ __forceinline__ void values8(uint32_t codes, uint32_t params, float (&x)[8])
{
    const float step = __uint_as_float(params << 16), low = __uint_as_float(params & 0xffff0000u);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fmaf(step, (float)((codes >> (4 * j)) & 15u), low);
}

// d = a * b + c with bf16 factors in the low halves of a and b, c in fp32.
__device__ __forceinline__ float fma_bf16(uint32_t a, uint32_t b, float c)
{
    float d;
    asm("{\n\t.reg .b16 a, b;\n\tcvt.u16.u32 a, %1;\n\tcvt.u16.u32 b, %2;\n\t"
        "fma.rn.f32.bf16 %0, a, b, %3;\n\t}\n"
        : "=f"(d)
        : "r"(a), "r"(b), "f"(c));
    return d;
}

// low - 128 step of a pair of parameters (exact unless low is negligible or
// 2^15 times step), and from it the values of codes j and j + 4: a code in
// the low mantissa bits of the bf16 128 is the bf16 number 128 + code, so one
// mask makes the factors of two values.
__device__ __forceinline__ float base128(uint32_t params)
{
    return fma_bf16(0xc300, params, __uint_as_float(params & 0xffff0000u));
}
__device__ __forceinline__ float2 value2(uint32_t codes, int j, uint32_t params, float base)
{
    uint32_t c;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(c) : "r"(codes >> (4 * j)));
    float2 x;
    asm("{\n\t.reg .b16 a, b, s, u;\n\tmov.b32 {a, b}, %2;\n\tmov.b32 {s, u}, %3;\n\t"
        "fma.rn.f32.bf16 %0, a, s, %4;\n\tfma.rn.f32.bf16 %1, b, s, %4;\n\t}\n"
        : "=f"(x.x), "=f"(x.y)
        : "r"(c), "r"(params), "f"(base));
    return x;
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
    int n, D, W, page_size, n_pages;
    uint8_t *pages;
    void *vk, *vv;
    int64_t ldv;
    int *status;
};

// One lane per 8 channels of a row (k and v); rows with a negative slot are
// left out.
template <typename T>
__global__ void __launch_bounds__(256) write_kernel(Write p)
{
    grid_dep_wait();  // programmatic dependent launch: inputs are ready
    grid_dep_launch();
    const int octs = p.D / 8;
    const int64_t total = (int64_t)p.n * octs;  // a multiple of 4: groups stay within a warp
    const int64_t stride = (int64_t)gridDim.x * blockDim.x;
    const int64_t first = (int64_t)blockIdx.x * blockDim.x + (threadIdx.x & ~31);
    for (int64_t base = first; base < total; base += stride) {
        const int64_t at = base + (threadIdx.x & 31);
        const bool in = at < total;
        const int row = in ? (int)(at / octs) : 0;
        const int ch = in ? (int)(at % octs) * 8 : 0;
        const int slot = in ? p.slots[row] : -1;
        const bool ok = slot >= 0 && slot < (int64_t)p.n_pages * p.page_size;
        float k[8] = {}, v[8] = {};
        if (ok) {
            load8(static_cast<const T *>(p.k) + row * p.ld + ch, k);
            load8(static_cast<const T *>(p.v) + row * p.ld + ch, v);
        } else if (slot >= 0 && ch == 0) {
            atomicOr(p.status, DC_DEVERR_PAGE);
        }
        float ks, kl, vs, vl;
        const uint32_t kc = quantise8(k, ks, kl), vc = quantise8(v, vs, vl);
        if (!ok) continue;
        const uint32_t kp = pack_params(ks, kl), vp = pack_params(vs, vl);
        uint8_t *rec = p.pages + record(slot / p.page_size, slot % p.page_size, ch / p.W, p.D / p.W,
                                        p.page_size, p.W);
        const int c = ch % p.W;
        *reinterpret_cast<uint2 *>(rec + c) = make_uint2(kc, vc);
        if (c % 32 == 0) *reinterpret_cast<uint2 *>(rec + p.W + c / 4) = make_uint2(kp, vp);
        if (p.vk) {
            values8(kc, kp, k);
            values8(vc, vp, v);
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
    int shift;  // page_size = 1 << shift
    int w4;  // w's rows start on 16-byte boundaries
    void *Z;
    int64_t ldz;
    int *status;
    int *counter;  // [B * nslab], zero between launches
    float *part;   // [gridDim.x][2][3][W]
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

constexpr int kWarps = 4, kThreads = 32 * kWarps, kResident = 4;
constexpr int kRows = 8;  // history rows of a block: never split over pages

// Blocks of kRows rows that position t's history has; 0: inactive.
__device__ __forceinline__ int row_blocks(const Decode &p, int t)
{
    return t < 0 || t >= p.cap ? 0 : t / kRows + 1;
}

__device__ __forceinline__ void join(float &m, float &num, float &den, float m2, float num2, float den2)
{
    const float mx = fmax_nan(m, m2);
    if (mx == -INFINITY) return;
    const float a = ex2(m - mx), c = ex2(m2 - mx);
    num = num * a + num2 * c;
    den = den * a + den2 * c;
    m = mx;
}

// The history of a slab (W channels of one sequence) is read once, in blocks
// of kRows rows by W/8 lanes of 8 channels each; exponents are in base 2
// (k and w scaled by log2 e), and each channel keeps (ref, num, den) with
// num, den = sums of 2^(y - ref) v and 2^(y - ref) in fp32.
//
// Work split: the row blocks of all (sequence, slab) items, one after the
// other, are cut into equal shares of q blocks, one share a CTA, so ragged
// lengths balance and a long sequence spreads over many CTAs.  An item that
// several CTAs share is merged, in CTA order, by the last of them to finish.
template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads, kResident) decode_kernel(Decode p)
{
    grid_dep_wait();  // programmatic dependent launch: inputs are ready
    grid_dep_launch();
    constexpr int RPW = 32 / LPR;       // row blocks a warp reads at once
    constexpr int W = LPR * 8;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int sub = lane / LPR, oct = lane % LPR;
    __shared__ float part[kWarps][3][W];
    __shared__ int s_sum[kWarps], s_max[kWarps], s_b, s_first, s_last;

    // this CTA's share [u, u1) of the row blocks
    int sum = 0, most = 0;
    for (int b = tid; b < p.B; b += kThreads) {
        const int t = p.pos[b], nb = row_blocks(p, t);
        sum += nb;
        most = max(most, nb);
        if (nb == 0 && b % gridDim.x == blockIdx.x) {  // an inactive sequence
            if (t >= 0) atomicOr(p.status, DC_DEVERR_FULL);
            const float zero[8] = {};
            for (int c = 0; c < p.D; c += 8) store8(static_cast<T *>(p.Z) + b * p.ldz + c, zero);
        }
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) {
        s_sum[warp] = sum;
        s_max[warp] = most;
    }
    __syncthreads();
    sum = most = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
        sum += s_sum[k];
        most = max(most, s_max[k]);
    }
    const int64_t total = (int64_t)sum * p.nslab;
    const int q = (int)max((total + gridDim.x - 1) / gridDim.x, (int64_t)sqrtf((float)most) + 1);
    int64_t u = (int64_t)blockIdx.x * q;
    const int64_t u1 = min(total, u + q);
    if (u >= u1) return;
    // the sequence that unit u lies in: blocks before it, over all sequences
    const int target = (int)(u / p.nslab);
    int before = 0;
    for (int b0 = 0;; b0 += kThreads) {
        const int b = b0 + tid;
        const int nb = b < p.B ? row_blocks(p, p.pos[b]) : 0;
        int inc = nb;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        __syncthreads();
        if (lane == 31) s_sum[warp] = inc;
        if (tid == 0) s_b = -1;
        __syncthreads();
        int at = before, all = 0;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            if (k < warp) at += s_sum[k];
            all += s_sum[k];
        }
        if (nb && target >= at + inc - nb && target < at + inc) {
            s_b = b;
            s_first = at + inc - nb;
        }
        __syncthreads();
        before += all;
        if (s_b >= 0) break;  // total > target: some sequence holds it
    }
    int b = s_b;
    int t = p.pos[b], nb = row_blocks(p, t);
    int slab = (int)((u - (int64_t)s_first * p.nslab) / nb);
    int blk = (int)((u - (int64_t)s_first * p.nslab) % nb);

    for (bool first = true;; first = false) {
        const int n = (int)min((int64_t)(nb - blk), u1 - u);
        const int ch = slab * W + oct * 8;
        const int32_t *tab = p.table + b * p.ldtab;
        const T *row = static_cast<const T *>(p.qkv) + b * p.ldq;
        const float *w = p.w + (ch / p.hs) * p.wh + t * p.ldw;
        // channels j and j + 4 of the lane's 8 in pairs
        float2 ref[4], num[4], den[4];
        float low = -INFINITY;  // the smallest ref, -inf while one is unset
#pragma unroll
        for (int j = 0; j < 4; ++j) ref[j] = num[j] = den[j] = make_float2(0.f, 0.f);
        for (int k = warp * RPW + sub; k < n; k += kWarps * RPW) {
            const int i0 = (blk + k) * kRows;
            const int page = tab[i0 >> p.shift];
            const bool ok = page >= 0 && page < p.n_pages;
            if (!ok && oct == 0) atomicOr(p.status, DC_DEVERR_PAGE);
            const int rows = ok ? min(kRows, t - i0) : 0;  // rows stored before this call
            uint8_t *rec = p.pages + record(ok ? page : 0, i0 & (p.page_size - 1), slab, p.nslab, p.page_size, W);
            uint2 code[kRows], par[kRows];
            float wl[kRows];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                code[r] = par[r] = make_uint2(0, 0);
                if (r < rows) {
                    code[r] = *reinterpret_cast<const uint2 *>(rec + r * (W * 5 / 4) + oct * 8);
                    par[r] = *reinterpret_cast<const uint2 *>(rec + r * (W * 5 / 4) + W + oct / 4 * 8);
                }
            }
            if (rows == kRows && p.w4) {
                const float4 a = *reinterpret_cast<const float4 *>(w + i0), c = *reinterpret_cast<const float4 *>(w + i0 + 4);
                wl[0] = a.x; wl[1] = a.y; wl[2] = a.z; wl[3] = a.w;
                wl[4] = c.x; wl[5] = c.y; wl[6] = c.z; wl[7] = c.w;
            } else {
#pragma unroll
                for (int r = 0; r < kRows; ++r) wl[r] = r < rows || (ok && i0 + r == t) ? w[i0 + r] : -INFINITY;
            }
            if (rows < kRows && ok) {  // position t itself: quantise and append
                float x[8], st, lo;
                const uint32_t lanes = 0xfu << (lane & ~3);
                uint2 c, pr;
                load8(row + p.D + ch, x);
                c.x = quantise8(x, st, lo, lanes);
                pr.x = pack_params(st, lo);
                load8(row + 2 * p.D + ch, x);
                c.y = quantise8(x, st, lo, lanes);
                pr.y = pack_params(st, lo);
                *reinterpret_cast<uint2 *>(rec + rows * (W * 5 / 4) + oct * 8) = c;
                if (oct % 4 == 0) *reinterpret_cast<uint2 *>(rec + rows * (W * 5 / 4) + W + oct * 2) = pr;
#pragma unroll
                for (int r = 0; r < kRows; ++r)
                    if (r == rows) {
                        code[r] = c;
                        par[r] = pr;
                    }
            }
            // y = log2(e) (k + w), k = low + step * code
            float ka[kRows], va[kRows], top = -INFINITY;  // top: a bound on the block's y
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                wl[r] *= kLog2e;
                ka[r] = base128(par[r].x);
                va[r] = base128(par[r].y);
                top = fmax_nan(top, fmaf(fma_bf16(0x430f, par[r].x, ka[r]), kLog2e, wl[r]));
            }
            // terms up to 2^16 above a channel's ref are summed as they are;
            // else the refs rise to the largest exponents so far.  (Exponents
            // beyond the range of fp32 in base 2, as of a bias of -FLT_MAX,
            // count as its end.)
            if (!(low > -1e30f && top <= low + 16.f)) {
#pragma unroll
                for (int r = 0; r < kRows; ++r)
                    if (isinf(wl[r]) && ok && (r < rows || i0 + r == t) && !isinf(w[i0 + r]))
                        wl[r] = copysignf(3.4028234e38f, wl[r]);
                low = INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float2 mx, old;
                    old.x = mx.x = den[j].x == 0.f ? -INFINITY : ref[j].x;
                    old.y = mx.y = den[j].y == 0.f ? -INFINITY : ref[j].y;
#pragma unroll
                    for (int r = 0; r < kRows; ++r) {
                        const float2 y = __ffma2_rn(value2(code[r].x, j, par[r].x, ka[r]),
                                                    make_float2(kLog2e, kLog2e), make_float2(wl[r], wl[r]));
                        mx.x = fmax_nan(mx.x, y.x);
                        mx.y = fmax_nan(mx.y, y.y);
                    }
                    low = fminf(low, fminf(mx.x, mx.y));
                    auto raise = [](float mx, float old, float &ref, float &num, float &den) {
                        if (mx == -INFINITY) return;
                        const float scale = ex2(old - mx);
                        num *= scale;
                        den *= scale;
                        ref = mx;
                    };
                    raise(mx.x, old.x, ref[j].x, num[j].x, den[j].x);
                    raise(mx.y, old.y, ref[j].y, num[j].y, den[j].y);
                }
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float2 y = __ffma2_rn(value2(code[r].x, j, par[r].x, ka[r]), make_float2(kLog2e, kLog2e),
                                          make_float2(wl[r], wl[r]));
                    y = __fadd2_rn(y, make_float2(-ref[j].x, -ref[j].y));
                    const float2 e = make_float2(ex2(y.x), ex2(y.y));
                    num[j] = __ffma2_rn(e, value2(code[r].y, j, par[r].y, va[r]), num[j]);
                    den[j] = __fadd2_rn(den[j], e);
                }
        }
        // blocks of a warp, then warps
        float fr[8], fu[8], fe[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            fe[j] = j < 4 ? den[j & 3].x : den[j & 3].y;
            fu[j] = j < 4 ? num[j & 3].x : num[j & 3].y;
            fr[j] = fe[j] == 0.f ? -INFINITY : j < 4 ? ref[j & 3].x : ref[j & 3].y;
#pragma unroll
            for (int o = LPR; o < 32; o *= 2) {
                const float m2 = __shfl_xor_sync(0xffffffffu, fr[j], o);
                const float n2 = __shfl_xor_sync(0xffffffffu, fu[j], o);
                const float d2 = __shfl_xor_sync(0xffffffffu, fe[j], o);
                join(fr[j], fu[j], fe[j], m2, n2, d2);
            }
        }
        if (sub == 0) {
            store8(&part[warp][0][oct * 8], fr);
            store8(&part[warp][1][oct * 8], fu);
            store8(&part[warp][2][oct * 8], fe);
        }
        __syncthreads();
        constexpr int CPT = (W + kThreads - 1) / kThreads;  // channels a thread finishes
        float fm[CPT], fn[CPT], fd[CPT];
#pragma unroll
        for (int k = 0; k < CPT; ++k) {
            const int c = tid + k * kThreads;
            if (c >= W) continue;
            fm[k] = part[0][0][c];
            fn[k] = part[0][1][c];
            fd[k] = part[0][2][c];
#pragma unroll
            for (int g = 1; g < kWarps; ++g) join(fm[k], fn[k], fd[k], part[g][0][c], part[g][1][c], part[g][2][c]);
        }
        bool finish = n == nb;
        if (!finish) {  // shared with other CTAs
            float *mine = p.part + ((int64_t)blockIdx.x * 2 + !first) * 3 * W;
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
            const int64_t u_item = u - blk;
            const int j0 = (int)(u_item / q), j1 = (int)((u_item + nb - 1) / q);
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
                    const int c = tid + k * kThreads;
                    if (c >= W) continue;
                    fm[k] = -INFINITY;
                    fn[k] = fd[k] = 0.f;
                    for (int g = j0; g <= j1; ++g) {
                        // the item is CTA g's first unless it begins inside g's share
                        const float *src = p.part + ((int64_t)g * 2 + (u_item > (int64_t)g * q)) * 3 * W + c;
                        join(fm[k], fn[k], fd[k], __ldcg(src), __ldcg(src + W), __ldcg(src + 2 * W));
                    }
                }
            }
        }
        if (finish) {
#pragma unroll
            for (int k = 0; k < CPT; ++k) {
                const int c = tid + k * kThreads;
                if (c >= W) continue;
                const float qv = to_f<T>(row[slab * W + c]);
                static_cast<T *>(p.Z)[b * p.ldz + slab * W + c] =
                    from_f<T>(fd[k] == 0.f ? 0.f : sigm(qv) * (fn[k] / fd[k]));
            }
        }
        u += n;
        if (u >= u1) return;
        blk = 0;
        if (++slab == p.nslab) {
            slab = 0;
            do t = p.pos[++b];  // u < total: there is another active one
            while ((nb = row_blocks(p, t)) == 0);
        }
        __syncthreads();  // part is reused
    }
}

static int decode_grid() { return kResident * sm_count(); }

template <typename T>
static cudaError_t launch_decode(const Decode &p, cudaStream_t st)
{
    const dim3 grid((unsigned)decode_grid()), block(kThreads);
    switch (p.W) {
        case 256: return launch_pdl(decode_kernel<T, 32>, grid, block, 0, st, 1, p);
        case 128: return launch_pdl(decode_kernel<T, 16>, grid, block, 0, st, 1, p);
        case 64: return launch_pdl(decode_kernel<T, 8>, grid, block, 0, st, 1, p);
        default: return launch_pdl(decode_kernel<T, 4>, grid, block, 0, st, 1, p);
    }
}

static int check_pool(int D, int n_pages, int page_size)
{
    if (D <= 0 || D % 32) return fail(DC_ERR_INVALID, "D must be a positive multiple of 32 (got %d)", D);
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
    if (n < 0) return fail(DC_ERR_INVALID, "bad row count %d", n);
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
    p.n_pages = n_pages;
    p.pages = static_cast<uint8_t *>(pages);
    p.vk = values_k;
    p.vv = values_v;
    p.ldv = ldv;
    p.status = device_status_word();
    if (!p.status) return fail(DC_ERR_CUDA, "no device status word");
    cudaStream_t st = as_stream(stream);
    KernelTimer kt("kv4_write", st);
    const int64_t blocks = ((int64_t)n * (D / 8) + 255) / 256;
    const dim3 grid((unsigned)std::min<int64_t>(blocks, (int64_t)sm_count() * 64));
    DC_CUDA_TRY(dtype == DC_F32 ? launch_pdl(write_kernel<float>, grid, dim3(256), 0, st, 1, p)
                                : launch_pdl(write_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, 1, p));
    return DC_OK;
}

size_t dc_aft_decode4_workspace_size(int B, int D)
{
    const int W = D > 0 ? kv4::slab_width(D) : 0;
    if (B <= 0 || !W) return 0;
    return round_up((int64_t)B * (D / W) * sizeof(int), 256) + (size_t)kv4::decode_grid() * 2 * 3 * W * sizeof(float);
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
    p.W = slab_width(D);
    p.nslab = D / p.W;
    p.n_pages = n_pages;
    p.page_size = page_size;
    p.cap = (int)std::min<int64_t>(Tmax, (int64_t)ldtab * page_size);
    for (p.shift = 3; 1 << p.shift < page_size;) ++p.shift;
    p.w4 = aligned16(w) && ldw % 4 == 0 && head_stride_w % 4 == 0;
    p.counter = static_cast<int *>(workspace);
    p.part = reinterpret_cast<float *>(static_cast<char *>(workspace) +
                                       round_up((int64_t)B * p.nslab * sizeof(int), 256));
    p.Z = Z;
    p.ldz = ldz;
    p.status = device_status_word();
    if (!p.status) return fail(DC_ERR_CUDA, "no device status word");
    if ((int64_t)B * (p.cap / kRows + 1) > INT32_MAX || (int64_t)B * p.nslab > INT32_MAX / 4)
        return fail(DC_ERR_INVALID, "B * Tmax or B * D too large");
    cudaStream_t st = as_stream(stream);
    KernelTimer kt("aft_decode4", st);
    DC_CUDA_TRY(dtype == DC_F32 ? launch_decode<float>(p, st) : launch_decode<__nv_bfloat16>(p, st));
    return DC_OK;
}

}  // extern "C"
