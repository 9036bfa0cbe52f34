/*
 * attn_pages_select.hip - which blocks of a long sequence a token attends:
 *
 *   bounds_kernel  a page's key bounds, per KV head and dimension
 *   score_kernel   each block's score, max over the group's heads of
 *                  sum_d q_d (q_d > 0 ? hi_d : lo_d): no key of the block can
 *                  give a larger q . k
 *   pick_kernel    the n_sel largest of a KV head, in the blocks' order
 *
 * A score is summed in double and rounded once: the order of the sum then
 * decides a choice in no case worth counting (a relative 2^-50 of two
 * neighbouring scores), where an f32 sum's order would decide one in some
 * thousand. The products are exact (24 x 11 bits).
 */
#include <math.h>
#include <stdint.h>

#include <hip/hip_runtime.h>

#include "attn_pages.h"

#pragma clang fp contract(off)

namespace janas {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef int16_t s8 __attribute__((ext_vector_type(8)));
typedef int8_t b8 __attribute__((ext_vector_type(8)));

constexpr float kHalfMax = 65504.0f;

/* x as a half that is not below it (up) or above it, within the halves' range */
__device__ __forceinline__ _Float16 outward(float x, bool up)
{
    x = fminf(fmaxf(x, -kHalfMax), kHalfMax);
    _Float16 h = (_Float16)x;
    if (up ? (float)h < x : (float)h > x) {
        uint16_t b = __builtin_bit_cast(uint16_t, h);
        if ((b & 0x7FFF) == 0)
            b = up ? 0x0001 : 0x8001;
        else if (up == !(b & 0x8000))
            b++;
        else
            b--;
        h = __builtin_bit_cast(_Float16, b);
    }
    return h;
}

/* 8 numbers of a cached row */
__device__ __forceinline__ void load8(int kv, const void *p, size_t at, float z, float *x)
{
    if (kv == kI8) {
        const b8 r = *(const b8 *)((const int8_t *)p + at);
#pragma unroll
        for (int e = 0; e < 8; e++)
            x[e] = (float)r[e] * z;
    } else if (kv == kI16) {
        const s8 r = *(const s8 *)((const int16_t *)p + at);
#pragma unroll
        for (int e = 0; e < 8; e++)
            x[e] = (float)r[e] * z;
    } else if (kv == kF16) {
        const h8 r = *(const h8 *)((const _Float16 *)p + at);
#pragma unroll
        for (int e = 0; e < 8; e++)
            x[e] = (float)r[e];
    } else {
        const f4 a = *(const f4 *)((const float *)p + at), b = *(const f4 *)((const float *)p + at + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[e] = a[e];
            x[4 + e] = b[e];
        }
    }
}

/*
 * A workgroup takes one block of a sequence and one KV head: its threads take 8
 * columns of every (256 / (hd / 8))-th row, then the rows' groups are joined in
 * LDS. Bound by reading the page once.
 */
__global__ __launch_bounds__(256) void bounds_kernel(const BoundsArgs A)
{
    __shared__ float sLo[256][8], sHi[256][8];
    const uint32_t tid = threadIdx.x, si = blockIdx.z, kvh = blockIdx.y;
    const uint32_t page = 1u << A.page_log, cap = A.max_pages << A.page_log;
    const uint32_t len = A.len[si] < cap ? A.len[si] : cap;
    uint32_t fresh = A.n_new ? A.n_new[si] : len;
    fresh = fresh < len ? fresh : len;
    if (fresh == 0)
        return;
    const uint32_t b1 = (len + page - 1) >> A.page_log, units = A.hd / 8, groups = 256 / units;
    const uint32_t u = tid % units, rg = tid / units;
    for (uint32_t b = ((len - fresh) >> A.page_log) + blockIdx.x; b < b1; b += gridDim.x) {
        const uint32_t pid = A.table[(size_t)si * A.max_pages + b];
        if (pid >= A.n_pages)
            continue;
        const uint32_t n = len - (b << A.page_log) < page ? len - (b << A.page_log) : page;
        const size_t row0 = ((size_t)pid * A.n_kv + kvh) << A.page_log;
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            lo[e] = INFINITY;
            hi[e] = -INFINITY;
        }
        if (rg < groups)
            for (uint32_t r = rg; r < n; r += groups) {
                float x[8];
                load8(A.kv, A.k, (row0 + r) * A.hd + 8 * u, A.ks ? A.ks[row0 + r] : 1.0f, x);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    lo[e] = fminf(lo[e], x[e]);
                    hi[e] = fmaxf(hi[e], x[e]);
                }
            }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            sLo[tid][e] = lo[e];
            sHi[tid][e] = hi[e];
        }
        __syncthreads();
        for (uint32_t c = tid; c < A.hd; c += 256) {
            float l = INFINITY, h = -INFINITY;
            for (uint32_t k = 0; k < groups; k++) {
                l = fminf(l, sLo[k * units + c / 8][c % 8]);
                h = fmaxf(h, sHi[k * units + c / 8][c % 8]);
            }
            _Float16 *const o = A.bounds + ((size_t)pid * A.n_kv + kvh) * 2 * A.hd;
            o[c] = outward(l, false);
            o[A.hd + c] = outward(h, true);
        }
        __syncthreads();
    }
}

/* a sequence's blocks in sight: [b0, b0 + n) */
struct Blocks {
    uint32_t b0, n;
};
__device__ __forceinline__ Blocks blocks_in_sight(const SelectArgs &A, const SeqView &s)
{
    const uint32_t page = 1u << A.page_log;
    if (!s.part || s.bad || s.end <= s.lo)
        return Blocks{0, 0};
    const uint32_t b0 = s.lo >> A.page_log;
    return Blocks{b0, ((s.end + page - 1) >> A.page_log) - b0};
}

__device__ __forceinline__ double sum16(double x)
{
#pragma unroll
    for (int o = 1; o < 16; o <<= 1)
        x += __shfl_xor(x, o, 64);
    return x;
}

constexpr uint32_t kScoreBlocks = 16;  /* blocks a workgroup at once, 16 lanes each */

__global__ __launch_bounds__(256) void score_kernel(const SelectArgs A)
{
    const uint32_t tid = threadIdx.x, si = blockIdx.z, kvh = blockIdx.y;
    const SeqView sv = seq_view(A, si);
    const Blocks bl = blocks_in_sight(A, sv);
    if (bl.n <= A.n_sel)
        return; /* all of them */
    const uint32_t c = tid % 16, hd = A.hd;
    const float *const q = A.q + (size_t)sv.row * A.q_stride + (size_t)kvh * A.group * hd;
    float *const out = A.score + ((size_t)si * A.n_kv + kvh) * A.max_pages;
    for (uint32_t j = blockIdx.x * kScoreBlocks + tid / 16; j < bl.n; j += gridDim.x * kScoreBlocks) {
        uint32_t pid = A.table[(size_t)si * A.max_pages + bl.b0 + j];
        pid = pid < A.n_pages ? pid : 0;
        const _Float16 *const box = A.bounds + ((size_t)pid * A.n_kv + kvh) * 2 * hd;
        float best = -INFINITY;
        for (uint32_t h = 0; h < A.group; h++) {
            double s = 0.0;
            for (uint32_t d = 8 * c; d < hd; d += 128) {
                const h8 lo = *(const h8 *)(box + d), hi = *(const h8 *)(box + hd + d);
                const float *const qd = q + (size_t)h * hd + d;
                const f4 qa = *(const f4 *)qd, qc = *(const f4 *)(qd + 4);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float x = e < 4 ? qa[e & 3] : qc[e & 3];
                    x = A.negate ? -x : x;
                    const float b = (float)(x > 0.0f ? hi[e] : lo[e]);
                    s = __builtin_fma((double)x, (double)b, s);
                }
            }
            best = fmaxf(best, (float)sum16(s));
        }
        if (c == 0)
            out[j] = best;
    }
}

constexpr uint32_t kPickThreads = 1024;
constexpr uint32_t kPickWaves = kPickThreads / 64;

/* a score's place in order, as a whole number above 0 */
__device__ __forceinline__ uint32_t score_key(float x)
{
    const uint32_t u = __float_as_uint(x + 0.0f); /* (-0 is 0) */
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return k == 0 ? 1 : k == 0xFFFFFFFFu ? 0xFFFFFFFEu : k;
}

/*
 * One workgroup a (sequence, KV head). The n_sel-th largest key is found 8 bits
 * at a time from the top (a histogram of the keys that share the bits found so
 * far); then the blocks above it, and of those at it the lowest, are written in
 * order by a running count.
 */
__global__ __launch_bounds__(kPickThreads) void pick_kernel(const SelectArgs A)
{
    __shared__ uint32_t sHist[256], sFound[2];
    __shared__ uint32_t sAbove[kPickWaves], sAt[kPickWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t kvh = blockIdx.x % A.n_kv, si = blockIdx.x / A.n_kv;
    const SeqView sv = seq_view(A, si);
    if (!sv.part)
        return;
    const Blocks bl = blocks_in_sight(A, sv);
    uint32_t *const sel = A.sel + ((size_t)si * A.n_kv + kvh) * A.n_sel;
    if (bl.n <= A.n_sel) {
        for (uint32_t i = tid; i < A.n_sel; i += kPickThreads)
            sel[i] = i < bl.n ? bl.b0 + i : kNone;
        return;
    }
    const float *const score = A.score + ((size_t)si * A.n_kv + kvh) * A.max_pages;
    /* the forced ones above every other */
    auto key = [&](uint32_t j) {
        return j < A.first || j >= bl.n - A.last ? 0xFFFFFFFFu : score_key(score[j]);
    };
    uint32_t found = 0, mask = 0, want = A.n_sel;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256)
            sHist[tid] = 0;
        __syncthreads();
        for (uint32_t j = tid; j < bl.n; j += kPickThreads) {
            const uint32_t k = key(j);
            if ((k & mask) == found)
                atomicAdd(&sHist[k >> shift & 255], 1u);
        }
        __syncthreads();
        /* the bin that holds the want-th from the top: one wave, 4 bins a lane
           from the top bin down */
        if (w == 0) {
            uint32_t n[4], sum = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                n[e] = sHist[255 - (4 * lane + e)];
                sum += n[e];
            }
            uint32_t s = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = __shfl_up(s, o, 64);
                s += lane >= (uint32_t)o ? y : 0;
            }
            uint32_t before = s - sum;
            if (before < want && want <= s) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (before < want && want <= before + n[e]) {
                        sFound[0] = 255 - (4 * lane + e);
                        sFound[1] = want - before;
                    }
                    before += n[e];
                }
            }
        }
        __syncthreads();
        found |= sFound[0] << shift;
        want = sFound[1];
        mask |= 255u << shift;
        __syncthreads();
    }
    /* `found` is the n_sel-th key; `want` of those equal to it are taken */
    uint32_t above = 0, at = 0; /* blocks above it and at it before this round */
    for (uint32_t j0 = 0; j0 < bl.n; j0 += kPickThreads) {
        const uint32_t j = j0 + tid;
        const uint32_t k = j < bl.n ? key(j) : 0;
        const uint64_t ma = __ballot(k > found), me = __ballot(k == found);
        if (lane == 0) {
            sAbove[w] = __popcll(ma);
            sAt[w] = __popcll(me);
        }
        __syncthreads();
        uint32_t na = above, ne = at;
        for (uint32_t i = 0; i < kPickWaves; i++) {
            na += i < w ? sAbove[i] : 0;
            ne += i < w ? sAt[i] : 0;
            above += sAbove[i];
            at += sAt[i];
        }
        __syncthreads();
        const uint64_t below = (1ull << lane) - 1;
        na += __popcll(ma & below);
        ne += __popcll(me & below);
        if (k > found || (k == found && k && ne < want))
            sel[na + (ne < want ? ne : want)] = bl.b0 + j;
    }
}

}  // namespace

hipError_t launch_bounds(const BoundsArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL(bounds_kernel, dim3(a.max_blocks, a.n_kv, a.n_seqs), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_select(const SelectArgs &a, hipStream_t s)
{
    /* as many workgroups as hold the table's blocks once, no more than fill
       the device eight times (max_pages may be far above the lengths) */
    const uint32_t pairs = a.n_seqs * a.n_kv;
    uint32_t x = (a.max_pages + kScoreBlocks - 1) / kScoreBlocks;
    const uint32_t most = pairs < 8 * a.cus ? 8 * a.cus / pairs : 1;
    x = x < most ? x : most;
    hipLaunchKernelGGL(score_kernel, dim3(x, a.n_kv, a.n_seqs), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return e;
    hipLaunchKernelGGL(pick_kernel, dim3(pairs), dim3(kPickThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace janas
