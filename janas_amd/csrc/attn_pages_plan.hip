/*
 * attn_pages_plan.hip - a serving step's pages and slots from the sequences'
 * lengths, on the device: which free page each new block gets, and where each
 * packed token's row goes.
 *
 * Two sums over the sequences decide everything: the tokens before a sequence
 * (its first packed row) and the pages asked for before it (where in the stack
 * of free pages its own begin). One workgroup takes them, 64 or 1024 sequences
 * at a time, and for a small step (a decode's) writes tables and slots too: one
 * launch. A large step's tokens and pages go to a second kernel, a thread each,
 * which finds a token's sequence in the first rows by halving.
 *
 * Bound by its launches: a step of 48 sequences moves 2 KB (3.0 to 4.0 us, as an
 * empty kernel), one of 46 prompts and 44 000 tokens 0.56 MB (4.8 + 3.8 us).
 */
#include <stdint.h>

#include <hip/hip_runtime.h>

#include "attn_elem.h"
#include "attn_pages.h"

namespace janas {
namespace {

/* the sum of x (below 2^32) over the threads before this one; total: over all */
template <uint32_t WAVES>
__device__ __forceinline__ uint64_t scan_group(uint32_t x, uint64_t *lds, uint64_t &total)
{
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    /* (64 lanes: in halves) */
    const uint64_t s = (uint64_t)scan_wave(x >> 16) * 65536 + scan_wave(x & 0xFFFF);
    if constexpr (WAVES == 1) {
        total = (uint64_t)__builtin_amdgcn_readlane((uint32_t)(s >> 32), 63) << 32 |
                __builtin_amdgcn_readlane((uint32_t)s, 63);
        return s - x;
    }
    if (lane == 63)
        lds[w] = s;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (uint32_t i = 0; i < WAVES; i++) {
        const uint64_t y = lds[i];
        before += i < w ? y : 0;
        total += y;
    }
    __syncthreads();
    return before + s - x;
}

__device__ __forceinline__ uint64_t blocks_of(uint64_t positions, uint32_t page_log)
{
    return (positions + (1u << page_log) - 1) >> page_log;
}

/* the page that is k-th from the top of a stack of `top` (0: outside it, never
   read: a stack's count is checked against what is taken) */
__device__ __forceinline__ uint32_t stack_page(const PlanArgs &A, uint64_t top, uint64_t k)
{
    return k < top ? A.free_pages[top - 1 - k] : 0;
}

/* position p's slot in its page; none where the table or the stack names a page
   outside the pool, whose slots in 32 bits could be another page's */
__device__ __forceinline__ uint32_t slot_of(const PlanArgs &A, uint32_t page, uint32_t p)
{
    return page < A.n_pages ? (page << A.page_log) + (p & ((1u << A.page_log) - 1)) : kNone;
}

/* the last i of n with at[i] <= x (at[0] = 0) */
__device__ __forceinline__ uint32_t last_at(const uint32_t *at, uint32_t n, uint32_t x)
{
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (at[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

/*
 * WAVES x 64 sequences at a time. A step of a token or none for each of up to 64
 * takes one wave, whose scans need no LDS: what is left of its time is a launch
 * and two round trips, the counts and the pages (8.4 -> 3.0 us for 48 sequences,
 * against 16 waves).
 */
template <uint32_t WAVES>
__global__ __launch_bounds__(WAVES * 64) void plan_kernel(const PlanArgs A)
{
    constexpr uint32_t THREADS = WAVES * 64;
    __shared__ uint64_t sScan[WAVES];
    __shared__ uint32_t sOld[THREADS], sNew[THREADS], sNeed[THREADS], sTok[THREADS], sOk[THREADS];
    __shared__ uint64_t sTake[THREADS];
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint64_t room = (uint64_t)A.max_pages << A.page_log;
    uint64_t top = *A.n_free;
    /* the first THREADS sequences' */
    const uint32_t new0 = tid < A.n_seqs ? A.n_new[tid] : 0;
    const uint32_t len0 = tid < A.n_seqs ? A.len[tid] : 0;
    top = top < A.n_pages ? top : A.n_pages;
    /* every thread has the count before one of them may change it */
    __syncthreads();

    /* ---- released pages onto the stack, sequence after sequence ---- */
    for (uint32_t i0 = 0; i0 < A.n_seqs; i0 += THREADS) {
        const uint32_t i = i0 + tid;
        const bool gone = i < A.n_seqs && (i0 ? A.n_new[i] : new0) == kRelease;
        if (!__syncthreads_or(gone))
            continue;
        uint64_t all;
        uint32_t gave = 0;
        if (gone) {
            const uint64_t b = blocks_of(A.len[i], A.page_log);
            gave = b < A.max_pages ? (uint32_t)b : A.max_pages;
        }
        /* where each one's begin among them; then a thread a page (4 at a time: the
           reads before the writes), its sequence found by halving */
        const uint64_t at = scan_group<WAVES>(gave, sScan, all);
        sTok[tid] = at < 0xFFFFFFFFu ? (uint32_t)at : 0xFFFFFFFFu;
        __syncthreads();
        const uint32_t n = A.n_seqs - i0 < THREADS ? A.n_seqs - i0 : THREADS;
        /* (what the stack has room for: all, unless a page is in two places) */
        const uint32_t fit = (uint32_t)(all < A.n_pages - top ? all : A.n_pages - top);
        for (uint32_t f0 = tid; f0 < fit; f0 += 4 * THREADS) {
            uint32_t page[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint32_t f = f0 + e * THREADS < fit ? f0 + e * THREADS : fit - 1;
                const uint32_t k = last_at(sTok, n, f);
                page[e] = A.table[(size_t)(i0 + k) * A.max_pages + (f - sTok[k])];
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; e++)
                if (f0 + e * THREADS < fit)
                    A.free_pages[top + f0 + e * THREADS] = page[e];
        }
        top += all;
        top = top < A.n_pages ? top : A.n_pages;
        /* what was pushed is read below, by other threads */
        __threadfence_block();
        __syncthreads();
    }

    /* ---- tokens and pages ---- */
    uint64_t tok = 0, asked = 0, took = 0;
    for (uint32_t i0 = 0; i0 < A.n_seqs; i0 += THREADS) {
        const uint32_t i = i0 + tid;
        const bool mine = i < A.n_seqs;
        uint32_t old = 0, add = 0;
        uint64_t all_tok, all_need;
        if (mine) {
            old = i0 ? A.len[i] : len0;
            add = i0 ? A.n_new[i] : new0;
            if (add == kRelease)
                old = add = 0;
        }
        const uint64_t first = tok + scan_group<WAVES>(add, sScan, all_tok);
        const bool fits = (uint64_t)old + add <= room && first + add <= A.max_tokens;
        const uint32_t have = (uint32_t)blocks_of(old, A.page_log);
        const uint32_t held = (uint32_t)blocks_of((uint64_t)old + add, A.page_log);
        const uint32_t need = fits ? held - have : 0;
        const uint64_t before = asked + scan_group<WAVES>(need, sScan, all_need);
        const bool ok = fits && (need == 0 || before + need <= top);
        /* the pages taken up to here: once a sequence found too few, none */
        uint64_t take = before;
        uint64_t all_take = all_need;
        if (asked + all_need > top)
            take = took + scan_group<WAVES>(ok ? need : 0, sScan, all_take);
        const bool many = mine && (add > 1 || need > 1);
        if (A.whole && mine && !many) {
            /* a token or none, a page or none */
            uint32_t *const row = A.table + (size_t)i * A.max_pages;
            uint32_t page = 0;
            if (ok && add)
                page = need ? stack_page(A, top, take) : row[old >> A.page_log];
            if (ok && need)
                row[have] = page;
            if (add && first < A.max_tokens) {
                const uint32_t s = ok ? slot_of(A, page, old) : kNone;
                A.slot[first] = s;
                A.pos[first] = s != kNone ? old : 0;
                A.seq[first] = i;
            }
        }
        if (mine) {
            A.start[i] = first < 0xFFFFFFFFu ? (uint32_t)first : 0xFFFFFFFFu;
            A.taken[i] = (uint32_t)take;
            A.granted[i] = ok ? add : 0;
            A.len_out[i] = old + (ok ? add : 0);
        }
        if (A.whole && __syncthreads_or(many)) {
            /* the others, a wave a sequence */
            sOld[tid] = old;
            sNew[tid] = many ? (add < A.max_tokens ? add : A.max_tokens) : 0;
            sNeed[tid] = many && ok ? need : 0;
            sTok[tid] = first < A.max_tokens ? (uint32_t)first : A.max_tokens;
            sTake[tid] = take;
            sOk[tid] = ok;
            __syncthreads();
            for (uint32_t k = w; k < THREADS && i0 + k < A.n_seqs; k += WAVES) {
                const uint32_t n = sNew[k], q = sNeed[k], at = sTok[k], o = sOld[k];
                const uint32_t h = (uint32_t)blocks_of(o, A.page_log);
                uint32_t *const row = A.table + (size_t)(i0 + k) * A.max_pages;
                for (uint32_t b = lane; b < q; b += 64)
                    row[h + b] = stack_page(A, top, sTake[k] + b);
                for (uint32_t t = lane; t < n && at + t < A.max_tokens; t += 64) {
                    uint32_t s = kNone, p = 0;
                    if (sOk[k]) {
                        p = o + t;
                        const uint32_t b = p >> A.page_log;
                        s = b < h ? row[b] : stack_page(A, top, sTake[k] + b - h);
                        s = slot_of(A, s, p);
                    }
                    A.slot[at + t] = s;
                    A.pos[at + t] = s != kNone ? p : 0;
                    A.seq[at + t] = i0 + k;
                }
            }
            __syncthreads();
        }
        tok += all_tok;
        asked += all_need;
        took += all_take;
    }
    if (tid == 0) {
        A.start[A.n_seqs] = tok < 0xFFFFFFFFu ? (uint32_t)tok : 0xFFFFFFFFu;
        A.taken[A.n_seqs] = (uint32_t)took;
        *A.n_free_out = (uint32_t)(top - took);
    }
    if (A.whole)
        for (uint64_t t = tok + tid; t < A.max_tokens; t += THREADS) {
            A.slot[t] = kNone;
            A.pos[t] = A.seq[t] = 0;
        }
}

/* The tables' and the tokens' part of a large step: workgroups of 256 threads,
   the first n_tok of them over tokens, the rest over taken pages. It reads
   what plan_kernel left; a new block's page comes from the stack, not from the
   table, which other workgroups write. */
constexpr uint32_t kFillSeqs = 1024;   /* sequences whose sums fit LDS */

__global__ __launch_bounds__(256) void plan_fill_kernel(const PlanArgs A, uint32_t n_tok)
{
    __shared__ uint32_t sAt[kFillSeqs];
    const bool pages = blockIdx.x >= n_tok;
    const uint32_t *at = pages ? A.taken : A.start;
    const uint32_t took = A.taken[A.n_seqs], tokens = A.start[A.n_seqs];
    const uint64_t top = (uint64_t)*A.n_free_out + took;
    if (A.n_seqs <= kFillSeqs) {
        for (uint32_t i = threadIdx.x; i < A.n_seqs; i += 256)
            sAt[i] = at[i];
        __syncthreads();
        at = sAt;
    }
    if (pages) {
        const uint32_t k = (blockIdx.x - n_tok) * 256 + threadIdx.x;
        if (k >= took)
            return;
        const uint32_t i = last_at(at, A.n_seqs, k);
        const uint32_t h = (uint32_t)blocks_of(A.len_out[i] - A.granted[i], A.page_log);
        A.table[(size_t)i * A.max_pages + h + (k - at[i])] = stack_page(A, top, k);
        return;
    }
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    if (t >= A.max_tokens)
        return;
    uint32_t s = kNone, p = 0, i = 0;
    if (t < tokens) {
        i = last_at(at, A.n_seqs, t);
        const uint32_t n = A.granted[i], end = A.len_out[i], take = A.taken[i];
        if (n) {
            const uint32_t old = end - n;
            const uint32_t h = (uint32_t)blocks_of(old, A.page_log);
            p = old + (t - at[i]);
            const uint32_t b = p >> A.page_log;
            s = b < h ? A.table[(size_t)i * A.max_pages + b]
                      : stack_page(A, top, (uint64_t)take + b - h);
            s = slot_of(A, s, p);
        }
    }
    A.slot[t] = s;
    A.pos[t] = s != kNone ? p : 0;
    A.seq[t] = i;
}

}  // namespace

hipError_t launch_plan(PlanArgs a, hipStream_t s)
{
    /* what the first kernel's waves write in about the time of a launch: a row or
       so a lane */
    a.whole = a.max_tokens <= (a.n_seqs <= 64 ? 256 : 4096);
    if (a.n_seqs <= 64 && a.whole)
        hipLaunchKernelGGL(plan_kernel<1>, dim3(1), dim3(64), 0, s, a);
    else if (a.n_seqs <= 256)
        hipLaunchKernelGGL(plan_kernel<4>, dim3(1), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(plan_kernel<16>, dim3(1), dim3(1024), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.whole)
        return e;
    const uint32_t n_tok = (a.max_tokens + 255) / 256;
    /* a sequence's tokens take at most a page each, and one more a sequence */
    uint64_t pages = ((uint64_t)a.max_tokens >> a.page_log) + a.n_seqs;
    pages = pages < a.n_pages ? pages : a.n_pages;
    const uint32_t n_page = (uint32_t)((pages + 255) / 256);
    hipLaunchKernelGGL(plan_fill_kernel, dim3(n_tok + n_page), dim3(256), 0, s, a, n_tok);
    return hipGetLastError();
}

}  // namespace janas
