// Kernels of a generation batch whose sequences have lengths of their own:
//
//   page_tables       block tables and slot maps from request lengths
//   logits_controls   penalties for repeated tokens, biases, grammar masks
//   greedy_embed_rows argmax and next embedding, a position per row
//
// The reference samples on the host, one sequence at a time, after copying
// the logits back (example/bin/shakespear4.dart:176-216) and has none of
// these.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "dc_internal.h"
#include "dc_ptx.cuh"

namespace dc {
namespace ragged {

constexpr int DC_DEVERR_INDEX = 0x20;   // a token id outside [0, V)
constexpr int DC_DEVERR_FULL = 0x40;    // decode ran past the sequence capacity
constexpr int DC_DEVERR_POOL = 0x100;   // no page for a token: free list or table row used up

// ------------------------------------------------------------ page tables
// Request b has start tokens in pages listed in its table row and gets count
// more: have = ceil(start / ps) pages are there, last = ceil((start + count) /
// ps) (at most the row's length) are needed, and the missing ones are taken
// from the free list in request order, at head + the sum of what earlier
// requests take.  Every page is thus known by arithmetic from two prefix
// sums, so table entries and slots are written independently of each other,
// by as many CTAs as there is work for.
constexpr int kTabThreads = 1024;

struct Tables {
    const int32_t *start, *count;
    int B, shift;
    const int32_t *free_pages;
    int n_free;
    const int32_t *head;
    int32_t *head_out, *table;
    int ldtab;
    int32_t *slots;
    int n_slots, ld_slots;
    int slots4;  // slots is 16-byte aligned
    int32_t *row_start;
    int *status;
};

// Exclusive prefix sums of two values over the block, and their totals.
__device__ __forceinline__ void scan2(int64_t &a, int &b, int64_t &ta, int &tb)
{
    __shared__ int64_t wa[32];
    __shared__ int wb[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t ia = a;
    int ib = b;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int64_t ua = __shfl_up_sync(0xffffffffu, ia, o);
        const int ub = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) {
            ia += ua;
            ib += ub;
        }
    }
    __syncthreads();
    if (lane == 31) {
        wa[warp] = ia;
        wb[warp] = ib;
    }
    __syncthreads();
    int64_t sa = lane < (int)(blockDim.x >> 5) ? wa[lane] : 0;
    int sb = lane < (int)(blockDim.x >> 5) ? wb[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int64_t ua = __shfl_up_sync(0xffffffffu, sa, o);
        const int ub = __shfl_up_sync(0xffffffffu, sb, o);
        if (lane >= o) {
            sa += ua;
            sb += ub;
        }
    }
    ta = __shfl_sync(0xffffffffu, sa, 31);
    tb = __shfl_sync(0xffffffffu, sb, 31);
    const int64_t before_a = __shfl_sync(0xffffffffu, sa, (warp + 31) & 31);
    const int before_b = __shfl_sync(0xffffffffu, sb, (warp + 31) & 31);
    a = ia - a + (warp ? before_a : 0);
    b = ib - b + (warp ? before_b : 0);
}

// Every CTA finds the prefix sums (rounds of kTabThreads requests) and writes
// its part of the table entries and slots, up to four slots a thread.  Latency-bound:
// the chain is lengths, two prefix sums, free pages, stores (64 requests of
// one token 4.0 us, 500 prompts of 1024 tokens on average 6.4 us).
__global__ void __launch_bounds__(kTabThreads) tables_kernel(const __grid_constant__ Tables p)
{
    grid_dep_wait();  // programmatic dependent launch: inputs are ready
    grid_dep_launch();
    // requests of this round: first token, tokens, pages there and needed,
    // free page of table column 0 (column c >= have takes free[base + c]),
    // packed row (none counts behind the slots)
    __shared__ int s_start[kTabThreads], s_count[kTabThreads], s_have[kTabThreads], s_last[kTabThreads],
        s_base[kTabThreads], s_row[kTabThreads + 1];
    const int ps = 1 << p.shift, tid = threadIdx.x;
    const int64_t thread = (int64_t)blockIdx.x * kTabThreads + tid, threads = (int64_t)gridDim.x * kTabThreads;
    const int head = min(max(0, *p.head), p.n_free);
    int64_t rows = 0;
    int pages = 0, err = 0;
    auto clip = [&](int64_t x) { return (int)min(x, (int64_t)INT32_MAX); };
    for (int b0 = 0; b0 < p.B; b0 += kTabThreads) {
        const int b = b0 + tid, nb = min(kTabThreads, p.B - b0);
        int start = 0, count = 0, have = 0, last = 0;
        if (b < p.B) {
            start = p.start[b];
            count = start < 0 ? 0 : max(0, p.count[b]);
            start = max(0, start);
            have = (int)(((int64_t)start + ps - 1) >> p.shift);
            const int64_t want = ((int64_t)start + count + ps - 1) >> p.shift;
            if (count && want > p.ldtab) err = 1;
            last = (int)min((int64_t)p.ldtab, want);
        }
        const int need = max(0, last - have);
        int64_t row = count, trow;
        int first = need, tpages;
        scan2(row, first, trow, tpages);
        s_start[tid] = start;
        s_count[tid] = count;
        s_have[tid] = have;
        s_last[tid] = last;
        s_row[tid] = clip(rows + row);
        s_base[tid] = (int)min((int64_t)INT32_MAX / 2, (int64_t)head + pages + first) - have;
        if (tid == 0) s_row[nb] = clip(rows + trow);
        if (b < p.B && p.row_start && blockIdx.x == 0) p.row_start[b] = clip(rows + row);
        if (need && (int64_t)head + pages + first + need > p.n_free) err = 1;
        __syncthreads();
        // table entries: a warp per request
        for (int r = (int)(thread >> 5); r < nb; r += (int)(threads >> 5)) {
            for (int c = s_have[r] + (tid & 31); c < s_last[r]; c += 32) {
                const int at = s_base[r] + c;
                p.table[(int64_t)(b0 + r) * p.ldtab + c] = at < p.n_free ? p.free_pages[at] : -1;
            }
        }
        // slots i0 .. i0+per-1 of [from, to); where(i, r, j): the request of
        // slot i and which of its tokens, or false
        auto write = [&](int64_t i0, int per, int64_t from, int64_t to, auto where) {
            int v[4], at_r = -1, at_c = -1, page = -1;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = -1;
                const int64_t i = i0 + k;
                int r, j;
                if (k >= per || i < from || i >= to || !where(i, r, j)) continue;
                const int64_t t = (int64_t)s_start[r] + j;
                if (t >> p.shift >= p.ldtab) continue;
                const int c = (int)(t >> p.shift);
                if (r != at_r || c != at_c) {  // another page than the last slot's
                    at_r = r;
                    at_c = c;
                    page = -1;
                    if (c < s_have[r])  // the page that start ends in
                        page = p.table[(int64_t)(b0 + r) * p.ldtab + c];
                    else if (s_base[r] + c < p.n_free)
                        page = p.free_pages[s_base[r] + c];
                }
                const int64_t slot = (int64_t)page * ps + (t & (ps - 1));
                if (page < 0 || slot > INT32_MAX)
                    err = 1;
                else
                    v[k] = (int)slot;
            }
            if (per == 4 && p.slots4 && i0 >= from && i0 + 4 <= to) {
                *reinterpret_cast<int4 *>(p.slots + i0) = make_int4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k < per && i0 + k >= from && i0 + k < to) p.slots[i0 + k] = v[k];
            }
        };
        // few slots: one a thread, so that their pages are read side by side
        auto per_thread = [&](int64_t n) { return n <= threads ? 1 : 4; };
        if (p.slots && p.ld_slots) {
            const int64_t from = (int64_t)b0 * p.ld_slots, to = (int64_t)(b0 + nb) * p.ld_slots;
            const int per = per_thread(to - from);
            for (int64_t i = (from & -per) + per * thread; i < to; i += per * threads)
                write(i, per, from, to, [&](int64_t i, int &r, int &j) {
                    const uint32_t d = (uint32_t)(i - from);  // below n_slots
                    r = (int)(d / (uint32_t)p.ld_slots);
                    j = (int)(d - (uint32_t)r * (uint32_t)p.ld_slots);
                    return j < s_count[r];
                });
            if (b < p.B && count > p.ld_slots) err = 1;
        } else if (p.slots) {
            const int64_t from = s_row[0], to = min(s_row[nb], p.n_slots);
            const int per = per_thread(to - from);
            for (int64_t i = (from & -per) + per * thread; i < to; i += per * threads) {
                int lo = 0, hi = nb - 1;  // last request that starts at or before the first slot
                const int64_t x = max(i, from);
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (s_row[mid] <= x) lo = mid;
                    else hi = mid - 1;
                }
                write(i, per, from, to, [&](int64_t i, int &r, int &j) {
                    while (lo + 1 < nb && s_row[lo + 1] <= i) ++lo;
                    r = lo;
                    j = (int)(i - s_row[lo]);
                    return true;
                });
            }
            if (s_row[nb] > p.n_slots) err = 1;
        }
        rows += trow;
        pages += tpages;
        __syncthreads();
    }
    if (p.slots) {  // behind the last token
        const int64_t used = p.ld_slots ? (int64_t)p.B * p.ld_slots : rows;
        for (int64_t i = used + thread; i < p.n_slots; i += threads) p.slots[i] = -1;
    }
    if (thread == 0) {
        if (p.row_start) p.row_start[p.B] = clip(rows);
        if (p.head_out) *p.head_out = (int)min((int64_t)p.n_free, (int64_t)head + pages);
    }
    if (err) atomicOr(p.status, DC_DEVERR_POOL);
}

// ------------------------------------------------------------ logits
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

struct Logits {
    const void *in;
    void *out;
    int64_t ldl, ldo;
    int B, V, chunk, chunks;
    const int32_t *tokens;
    int ldt;
    const int32_t *pos;
    int pos_stride;
    const int32_t *prompt;
    const float *rep, *pres, *freq, *bias;
    int64_t ldb;
    const uint32_t *mask;
    int64_t ldm;
};

constexpr uint32_t kSeen = 0x80000000u;
constexpr int kTile = 4;  // logits of a lane in flight

// One block per chunk of a row's vocabulary: the tokens known so far that
// fall into the chunk are counted in shared memory (bit 31: seen in the
// prompt; the rest: how often generated), then the logits stream through, a
// warp's lanes side by side so that rows of any alignment are read and
// written in whole lines.  A larger chunk scans the tokens less often, a
// smaller one spreads few rows over more SMs.  512 x 50257 bf16 logits, a bias
// and a mask a row, 2048 known tokens on average, take 49 us (213 MB, 0.67 of
// the measured copy rate): 41 us without penalties, the rest their arithmetic
// and the counting.  Four logits a lane in flight; eight and
// two were slower (60 us).
template <typename T>
__global__ void __launch_bounds__(512) logits_kernel(const __grid_constant__ Logits p)
{
    grid_dep_wait();  // programmatic dependent launch: inputs are ready
    grid_dep_launch();
    extern __shared__ __align__(16) uint32_t hist[];
    const int b = blockIdx.x / p.chunks, v0 = blockIdx.x % p.chunks * p.chunk;
    const int n = min(p.chunk, p.V - v0);  // chunk: a multiple of 32
    const bool pens = p.rep || p.pres || p.freq;
    if (pens) {
        // long chunks come into L2 while the tokens are counted (1000 x 32000
        // fp32: 58 -> 50 us; short ones would wait for the request: 64 x 8192
        // 3.2 -> 3.4 us).  Whole 16 bytes within the chunk.
        if (threadIdx.x == 0 && p.chunk > 8192) {
            const uintptr_t first = reinterpret_cast<uintptr_t>(static_cast<const T *>(p.in) + b * p.ldl + v0);
            const uintptr_t from = (first + 15) & ~uintptr_t(15), to = (first + n * sizeof(T)) & ~uintptr_t(15);
            if (from < to)
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"((uint32_t)(to - from)) : "memory");
        }
        for (int i = threadIdx.x; i < p.chunk / 4; i += blockDim.x)
            reinterpret_cast<uint4 *>(hist)[i] = make_uint4(0, 0, 0, 0);
        const int at = p.pos[(int64_t)b * p.pos_stride];
        const int known = at < 0 ? 0 : min(p.ldt - 1, at) + 1;
        const int prompt = p.prompt ? p.prompt[b] : 0;
        const int32_t *tok = p.tokens + (int64_t)b * p.ldt;
        __syncthreads();
        for (int i0 = threadIdx.x; i0 < known; i0 += 4 * blockDim.x) {
            int v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = i0 + k * (int)blockDim.x < known ? tok[i0 + k * blockDim.x] : -1;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t c = (uint32_t)v[k] - (uint32_t)v0;
                if (v[k] >= 0 && c < (uint32_t)n) {
                    if (i0 + k * (int)blockDim.x < prompt) atomicOr(hist + c, kSeen);
                    else atomicAdd(hist + c, 1u);
                }
            }
        }
        __syncthreads();
    }
    const float rep = p.rep ? p.rep[b] : 1.f, inv = 1.f / rep;
    const float pres = p.pres ? p.pres[b] : 0.f, freq = p.freq ? p.freq[b] : 0.f;
    const T *in = static_cast<const T *>(p.in) + b * p.ldl + v0;
    T *out = static_cast<T *>(p.out) + b * p.ldo + v0;
    const float *bias = p.bias ? p.bias + b * p.ldb + v0 : nullptr;
    const uint32_t *mask = p.mask ? p.mask + b * p.ldm + v0 / 32 : nullptr;
    const int lane = threadIdx.x & 31;
    auto tile = [&](int t0, auto whole) {  // logits t0 + 32 k + lane
        const int left = whole ? 32 * kTile : n - t0 - lane;
        const T *src = in + t0 + lane;
        T x[kTile];
        float y[kTile];
        uint32_t m[kTile], h[kTile];
#pragma unroll
        for (int k = 0; k < kTile; ++k) x[k] = whole || 32 * k < left ? src[32 * k] : from_f<T>(0.f);
        if (bias) {
            const float *add = bias + t0 + lane;
#pragma unroll
            for (int k = 0; k < kTile; ++k) y[k] = whole || 32 * k < left ? add[32 * k] : 0.f;
        }
        if (mask) {
            const uint32_t *word = mask + t0 / 32;
#pragma unroll
            for (int k = 0; k < kTile; ++k) m[k] = whole || 32 * k < left + lane ? word[k] : 0;
        }
        if (pens) {
            const uint32_t *seen = hist + t0 + lane;
#pragma unroll
            for (int k = 0; k < kTile; ++k) h[k] = whole || 32 * k < left ? seen[32 * k] : 0;
        }
        T *dst = out + t0 + lane;
#pragma unroll
        for (int k = 0; k < kTile; ++k) {
            float f = to_f<T>(x[k]);
            if (pens) {
                const float made = (float)(h[k] & ~kSeen), g = f * (f > 0.f ? inv : rep);
                if (h[k]) f = g;
                if (made > 0.f) f = fmaf(-freq, made, f) - pres;
            }
            if (bias) f += y[k];
            if (mask && !(m[k] >> lane & 1u)) f = -INFINITY;
            if (whole || 32 * k < left) dst[32 * k] = from_f<T>(f);
        }
    };
    int t0 = (threadIdx.x & ~31) * kTile;
    for (; t0 + 32 * kTile <= n; t0 += blockDim.x * kTile) tile(t0, std::true_type{});
    if (t0 < n) tile(t0, std::false_type{});
}

// ------------------------------------------------------------ pick
struct Pick {
    const void *logits;
    int64_t ldl;
    int B, V;
    const float *wte, *wpe;
    const int32_t *pos;
    int32_t *pos_out;
    int D;
    int32_t *tokens;
    int ldt;
    float *x;
    int *status;
    int cluster;  // blocks a row
};

// One block per row, or a cluster of them for few long rows: argmax (lowest
// index on ties, NaN never wins), the token's embedding at the row's next
// position, the advanced position.  64 bytes of a thread are in flight.  512
// rows of 50257 bf16 logits take 14.9 us (0.58 of the measured copy rate, one
// wave of blocks); loads of single logits took 18.4 us, two blocks a row 20.7.
template <typename T>
__global__ void __launch_bounds__(512) pick_kernel(const __grid_constant__ Pick p)
{
    grid_dep_wait();  // programmatic dependent launch: inputs are ready
    grid_dep_launch();
    __shared__ float sv[16];
    __shared__ int si[16];
    const int parts = p.cluster, b = blockIdx.x / parts, part = blockIdx.x % parts;
    const int at = p.pos[b];
    if (parts > 1) cluster_sync_all();  // pos_out may be pos: every thread has read its position
    else __syncthreads();
    if (at < 0 || at >= p.ldt - 1) {  // the same in the row's whole cluster
        if (part == 0 && threadIdx.x == 0) {
            p.pos_out[b] = at;
            if (at >= 0) atomicOr(p.status, DC_DEVERR_FULL);
        }
        return;
    }
    const T *l = static_cast<const T *>(p.logits) + b * p.ldl;
    float best = -INFINITY;
    int bi = INT_MAX;
    // whole 16-byte vectors, and the logits before and behind them one by one;
    // a thread meets its logits in increasing order
    constexpr int N = 16 / sizeof(T), U = 4;
    const int head = min(p.V, (int)((16 - (reinterpret_cast<uintptr_t>(l) & 15)) % 16 / sizeof(T)));
    const int vectors = (p.V - head) / N, tail = head + vectors * N;
    const uint4 *l4 = reinterpret_cast<const uint4 *>(l + head);
    auto single = [&](int v) {
        const float f = to_f<T>(l[v]);
        if (f > best || (f == best && bi == INT_MAX)) {
            best = f;
            bi = v;
        }
    };
    if (part == 0 && (int)threadIdx.x < head) single(threadIdx.x);
    const int step = blockDim.x * parts;
    for (int64_t i0 = part * blockDim.x + threadIdx.x; i0 < vectors; i0 += U * step) {
        uint4 x[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int64_t i = i0 + k * step;
            x[k] = l4[i < vectors ? i : i0];
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const T *e = reinterpret_cast<const T *>(&x[k]);
            float f[N], top = NAN;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                f[j] = to_f<T>(e[j]);
                top = fmaxf(top, f[j]);  // of the numbers among them
            }
            if (top > best || (top == best && bi == INT_MAX)) {  // a vector read again brings nothing
                best = top;
#pragma unroll
                for (int j = N - 1; j >= 0; --j)
                    if (f[j] == top) bi = head + (int)(i0 + k * step) * N + j;
            }
        }
    }
    if (part == 0 && tail + (int)threadIdx.x < p.V) single(tail + threadIdx.x);
    auto take = [&](float x, int v) {
        if (x > best || (x == best && v < bi)) {
            best = x;
            bi = v;
        }
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, best, o);
        const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
        take(ov, oi);
    }
    if ((threadIdx.x & 31) == 0) {
        sv[threadIdx.x >> 5] = best;
        si[threadIdx.x >> 5] = bi;
    }
    __syncthreads();
    for (int k = 0; k < (int)blockDim.x / 32; ++k) take(sv[k], si[k]);
    if (parts > 1) {
        __syncthreads();
        if (threadIdx.x == 0) {
            sv[0] = best;
            si[0] = bi;
        }
        cluster_sync_all();
        if (part == 0)
            for (int k = 1; k < parts; ++k)
                take(ld_dsmem_f32(smem_in_cta(smem_u32(sv), k)),
                     __float_as_int(ld_dsmem_f32(smem_in_cta(smem_u32(si), k))));
        cluster_sync_all();  // the others' shared memory stays until it is read
        if (part) return;
    }
    const int tok = bi < p.V ? bi : 0;  // all NaN: token 0
    if (threadIdx.x == 0) {
        p.tokens[(int64_t)b * p.ldt + at + 1] = tok;
        p.pos_out[b] = at + 1;
    }
    if (p.x) {
        const float *e = p.wte + (int64_t)tok * p.D, *q = p.wpe + (int64_t)(at + 1) * p.D;
        for (int d = threadIdx.x; d < p.D; d += blockDim.x) p.x[(int64_t)b * p.D + d] = e[d] + q[d];
    }
}

}  // namespace ragged
}  // namespace dc

using namespace dc;
using namespace dc::ragged;

extern "C" {

int dc_page_tables(const int32_t *start, const int32_t *count, int B, int page_size, const int32_t *free_pages,
                   int n_free, const int32_t *free_head, int32_t *free_head_out, int32_t *table, int ldtab,
                   int32_t *slots, int n_slots, int ld_slots, int32_t *row_start, void *stream)
{
    clear_error();
    if (B < 0 || n_free < 0 || ldtab <= 0 || n_slots < 0 || ld_slots < 0)
        return fail(DC_ERR_INVALID, "bad shape B=%d n_free=%d ldtab=%d n_slots=%d ld_slots=%d", B, n_free, ldtab,
                    n_slots, ld_slots);
    if (page_size < 8 || page_size > 256 || (page_size & (page_size - 1)))
        return fail(DC_ERR_INVALID, "page_size must be 8, 16, 32, 64, 128 or 256 (got %d)", page_size);
    if ((int64_t)B * ldtab > INT32_MAX) return fail(DC_ERR_INVALID, "B * ldtab must be below 2^31");
    // the kernel's index into the free list is a sum of two of these
    if (n_free > INT32_MAX / 2 || ldtab > INT32_MAX / 2)
        return fail(DC_ERR_INVALID, "n_free and ldtab must be below 2^30");
    if (B == 0) return DC_OK;
    if (!start || !count || !free_pages || !free_head || !free_head_out || !table)
        return fail(DC_ERR_INVALID, "null pointer");
    if (slots && ld_slots && (int64_t)B * ld_slots > n_slots)
        return fail(DC_ERR_INVALID, "slots holds %d, B * ld_slots is %lld", n_slots, (long long)B * ld_slots);
    Tables p{};
    p.start = start;
    p.count = count;
    p.B = B;
    for (p.shift = 3; 1 << p.shift < page_size;) ++p.shift;
    p.free_pages = free_pages;
    p.n_free = n_free;
    p.head = free_head;
    p.head_out = free_head_out;
    p.table = table;
    p.ldtab = ldtab;
    p.slots = slots;
    p.n_slots = n_slots;
    p.ld_slots = ld_slots;
    p.row_start = row_start;
    p.status = device_status_word();
    if (!p.status) return fail(DC_ERR_CUDA, "no device status word");
    cudaStream_t st = as_stream(stream);
    KernelTimer kt("page_tables", st);
    p.slots4 = aligned16(slots);
    // A CTA per 1024 slots, or per 16 requests, up to one an SM (64 prompts of
    // 127 tokens: 5.0 us, per 4096 slots 6.2, on one CTA 6.8; 500 prompts of 1024
    // tokens: 6.4 us, on one CTA 504).  A head that is advanced in place takes
    // two launches then, and one CTA while that is faster.
    const int64_t room = slots ? n_slots : 0, work = std::max<int64_t>(room, (int64_t)64 * B);
    const bool in_place = free_head == free_head_out;
    const int grid = in_place && B <= kTabThreads && room <= 8192
                         ? 1 : (int)std::min<int64_t>(sm_count(), (work + 1023) / 1024);
    int last = grid;
    if (grid > 1 && in_place) {
        // other CTAs may still have to read the head that one would advance:
        // a second launch of one CTA does (and writes the same entries again)
        p.head_out = nullptr;
        DC_CUDA_TRY(launch_pdl(tables_kernel, dim3(grid), dim3(kTabThreads), 0, st, 1, p));
        p.head_out = free_head_out;
        p.slots = nullptr;
        p.row_start = nullptr;
        last = 1;
    }
    DC_CUDA_TRY(launch_pdl(tables_kernel, dim3(last), dim3(kTabThreads), 0, st, 1, p));
    return DC_OK;
}

int dc_logits_controls(const void *logits, int ldl, void *out, int ldo, int dtype, int B, int V,
                       const int32_t *tokens, int ldt, const int32_t *pos, int pos_stride,
                       const int32_t *prompt_len, const float *repetition, const float *presence,
                       const float *frequency, const float *bias, int ldb, const uint32_t *mask, int ldm,
                       void *stream)
{
    clear_error();
    if (B < 0 || V <= 0 || ldl < V || ldo < V) return fail(DC_ERR_INVALID, "bad shape B=%d V=%d", B, V);
    // the kernel steps through logits and tokens in 32 bits
    if (V >= 1 << 30 || ldt >= 1 << 30) return fail(DC_ERR_INVALID, "V and ldt must be below 2^30 (got %d, %d)", V, ldt);
    if (dtype != DC_F32 && dtype != DC_BF16) return fail(DC_ERR_INVALID, "bad dtype %d", dtype);
    if (B == 0) return DC_OK;
    if (!logits || !out) return fail(DC_ERR_INVALID, "null pointer");
    if (logits == out && ldl != ldo) return fail(DC_ERR_INVALID, "in place needs one row stride");
    const bool pens = repetition || presence || frequency;
    if (pens && (!tokens || !pos || ldt <= 0 || (pos_stride != 0 && pos_stride != 1)))
        return fail(DC_ERR_INVALID, "penalties need the tokens and positions (pos_stride 0 or 1)");
    if (bias && ldb != 0 && ldb < V) return fail(DC_ERR_INVALID, "ldb must be 0 (one bias) or at least V");
    if (mask && ldm != 0 && ldm < (V + 31) / 32)
        return fail(DC_ERR_INVALID, "ldm must be 0 (one mask) or at least ceil(V / 32)");
    Logits p{};
    p.in = logits;
    p.out = out;
    p.ldl = ldl;
    p.ldo = ldo;
    p.B = B;
    p.V = V;
    // chunks of 1024 while the grid is short of eight blocks an SM (64 x 32000
    // fp32: 6.3 us, four 7.4, twelve 7.2), of at most 16384 (64 KB of counts)
    const int64_t fill = (8LL * sm_count() + B - 1) / B;
    const int64_t want = std::max<int64_t>((V + 16383) / 16384, std::min<int64_t>((V + 1023) / 1024, fill));
    p.chunk = (int)round_up((V + want - 1) / want, 32);
    p.chunks = (V + p.chunk - 1) / p.chunk;
    p.tokens = tokens;
    p.ldt = ldt;
    p.pos = pos;
    p.pos_stride = pos_stride;
    p.prompt = prompt_len;
    p.rep = repetition;
    p.pres = presence;
    p.freq = frequency;
    p.bias = bias;
    p.ldb = ldb;
    p.mask = mask;
    p.ldm = ldm;
    if ((int64_t)B * p.chunks > INT32_MAX) return fail(DC_ERR_INVALID, "B * V too large");
    cudaStream_t st = as_stream(stream);
    KernelTimer kt("logits_controls", st);
    // long chunks leave room for few blocks an SM: more threads in each (64 x
    // 50257 in chunks of 2656: 256 threads 8.1 us, 512 10.4; 512 x 50257 in
    // chunks of 12576, one bias and mask: 512 threads 40 us, 256 50)
    const dim3 grid((unsigned)(B * p.chunks)), block(p.chunk > 8192 ? 512 : 256);
    const int smem = pens ? p.chunk * (int)sizeof(uint32_t) : 0;
    auto kernel = dtype == DC_F32 ? logits_kernel<float> : logits_kernel<__nv_bfloat16>;
    if (smem > 48 * 1024) {
        static SmemOnce once[2];
        DC_CUDA_TRY(once[dtype == DC_F32].set(kernel, 64 * 1024));
    }
    DC_CUDA_TRY(launch_pdl(kernel, grid, block, smem, st, 1, p));
    return DC_OK;
}

int dc_greedy_embed_rows(const void *logits, int ldl, int dtype, int B, int V, const float *wte,
                         const float *wpe, const int32_t *pos, int32_t *pos_out, int D, int32_t *tokens,
                         int ldt, float *x, void *stream)
{
    clear_error();
    if (B < 0 || V <= 0 || ldl < V || ldt <= 0) return fail(DC_ERR_INVALID, "bad shape B=%d V=%d ldt=%d", B, V, ldt);
    if (V >= 1 << 30) return fail(DC_ERR_INVALID, "V must be below 2^30 (got %d)", V);  // indices of 32 bits
    if (dtype != DC_F32 && dtype != DC_BF16) return fail(DC_ERR_INVALID, "bad dtype %d", dtype);
    if (B == 0) return DC_OK;
    if (!logits || !pos || !pos_out || !tokens) return fail(DC_ERR_INVALID, "null pointer");
    if (x && (!wte || !wpe || D <= 0)) return fail(DC_ERR_INVALID, "embedding tables needed");
    Pick p{};
    p.logits = logits;
    p.ldl = ldl;
    p.B = B;
    p.V = V;
    p.wte = wte;
    p.wpe = wpe;
    p.pos = pos;
    p.pos_out = pos_out;
    p.D = D;
    p.tokens = tokens;
    p.ldt = ldt;
    p.x = x;
    p.status = device_status_word();
    if (!p.status) return fail(DC_ERR_CUDA, "no device status word");
    cudaStream_t st = as_stream(stream);
    KernelTimer kt("greedy_embed_rows", st);
    // A cluster of 4 blocks a row while rows are few and long: rows of 131072
    // fp32 logits take 5.8 us instead of 9.1 (1 row), 9.7 instead of 16.2 (64);
    // at 32768 logits one block is as fast or faster (4.3 us both, against 4.4
    // and 5.3).
    // 8 blocks gain up to 1 us on one row and lose 3 us on 37.
    p.cluster = V >= 65536 && B <= sm_count() / 2 ? 4 : 1;
    // Fewer threads for short rows (64 x 2048: 256 threads 2.5 us, 512 2.65) and
    // for so many that blocks queue (512 x 512: 128 threads 3.0 us, 256 3.2, 512
    // 4.7; 512 x 8192: 256 threads 4.8 us, 512 6.2; 64 x 8192: 3.0 and 2.8).
    const int threads = 512 >> (V <= 2048) >> (V <= 16384 && B > 2 * sm_count());
    const dim3 grid((unsigned)(B * p.cluster)), block(threads);
    auto kernel = dtype == DC_F32 ? pick_kernel<float> : pick_kernel<__nv_bfloat16>;
    DC_CUDA_TRY(launch_pdl(kernel, grid, block, 0, st, p.cluster, p));
    return DC_OK;
}

}  // extern "C"
