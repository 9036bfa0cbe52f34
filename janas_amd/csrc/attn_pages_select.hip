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

#include "attn_elem.h"
#include "attn_pages.h"

#pragma clang fp contract(off)

namespace janas {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));
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

/* 8 numbers of a cached row as they are, and as floats */
template <int KV> struct Raw8;
template <> struct Raw8<kI8> { typedef b8 T; };
template <> struct Raw8<kI16> { typedef s8 T; };
template <> struct Raw8<kF16> { typedef h8 T; };
template <> struct Raw8<kF32> { typedef f8 T; };
template <int KV> __device__ __forceinline__ typename Raw8<KV>::T load8(const void *p, size_t at)
{
    typedef typename Raw8<KV>::T T;
    if constexpr (KV == kF32) { /* (aligned to 16 bytes) */
        const float *const x = (const float *)p + at;
        const f4 a = *(const f4 *)x, b = *(const f4 *)(x + 4);
        return T{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
        return *(const T *)((const char *)p + at * (sizeof(T) / 8));
    }
}

constexpr uint32_t kBoundRows = 4;     /* rows a thread asks for at once */

/*
 * A workgroup takes up to 128 columns of one block and KV head: its threads take 8
 * of them in every (256 / (columns / 8))-th row, four rows asked for at once (one
 * after the other: a page of 64 x 128 halves 5.1 -> 3.3 us, 5 x 6000 new positions
 * of 2 x 256 9.0 -> 7.2 us, 4.3 TB/s; 8 at once no faster), then the rows' groups are
 * joined in LDS. A workgroup for whole rows of 512 took 0.9 us longer. Bound by
 * reading the page once, and for a decode's one block by its chain of reads - length,
 * page, rows - and its launch.
 */
template <int KV> __global__ __launch_bounds__(256) void bounds_kernel(const BoundsArgs A)
{
    constexpr bool SCALED = KV == kI8 || KV == kI16;
    __shared__ __attribute__((aligned(16))) float sLo[256][8], sHi[256][8];
    const uint32_t tid = threadIdx.x, si = blockIdx.z, kvh = blockIdx.y;
    const uint32_t page = 1u << A.page_log, cap = A.max_pages << A.page_log;
    const uint32_t length = A.len[si], len = length < cap ? length : cap;
    uint32_t fresh = A.n_new ? A.n_new[si] : len;
    fresh = fresh < len ? fresh : len;
    if (fresh == 0)
        return;
    const uint32_t b1 = (len + page - 1) >> A.page_log;
    const uint32_t slices = bound_slices(A.hd), step = gridDim.x / slices;
    const uint32_t c0 = blockIdx.x % slices * kBoundCols;
    const uint32_t cols = A.hd - c0 < kBoundCols ? A.hd - c0 : kBoundCols;
    const uint32_t units = cols / 8, groups = 256 / units;
    const uint32_t u = tid % units, rg = tid / units;
    for (uint32_t b = ((len - fresh) >> A.page_log) + blockIdx.x / slices; b < b1; b += step) {
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
            for (uint32_t r0 = rg; r0 < n; r0 += kBoundRows * groups) {
                typename Raw8<KV>::T x[kBoundRows];
                float z[kBoundRows];
#pragma unroll
                for (uint32_t i = 0; i < kBoundRows; i++) {
                    /* (behind the last row: that one again) */
                    const uint32_t r = r0 + i * groups < n ? r0 + i * groups : n - 1;
                    x[i] = load8<KV>(A.k, (row0 + r) * A.hd + c0 + 8 * u);
                    z[i] = SCALED ? A.ks[row0 + r] : 1.0f;
                }
#pragma unroll
                for (uint32_t i = 0; i < kBoundRows; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float y = SCALED ? (float)x[i][e] * z[i] : (float)x[i][e];
                        lo[e] = fminf(lo[e], y);
                        hi[e] = fmaxf(hi[e], y);
                    }
            }
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            *(f4 *)&sLo[tid][e] = f4{lo[e], lo[e + 1], lo[e + 2], lo[e + 3]};
            *(f4 *)&sHi[tid][e] = f4{hi[e], hi[e + 1], hi[e + 2], hi[e + 3]};
        }
        __syncthreads();
        if (tid < cols) {
            const uint32_t c = tid;
            float l = INFINITY, h = -INFINITY;
#pragma unroll 8
            for (uint32_t k = 0; k < groups; k++) {
                l = fminf(l, sLo[k * units + c / 8][c % 8]);
                h = fmaxf(h, sHi[k * units + c / 8][c % 8]);
            }
            _Float16 *const o = A.bounds + ((size_t)pid * A.n_kv + kvh) * 2 * A.hd + c0;
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

template <int CTRL> __device__ __forceinline__ double dpp(double x)
{
    const uint2 u = __builtin_bit_cast(uint2, x);
    return __builtin_bit_cast(
        double, make_uint2(__builtin_amdgcn_update_dpp(0u, u.x, CTRL, 0xf, 0xf, false),
                           __builtin_amdgcn_update_dpp(0u, u.y, CTRL, 0xf, 0xf, false)));
}
/* one step of a sum over 16 lanes (CTRL pairs each lane with its partner) ... */
template <int CTRL> __device__ __forceinline__ double step(double x) { return x + dpp<CTRL>(x); }
/* ... and of two sums at once: the lanes with `hi` go on with b, the others with
   a */
template <int CTRL> __device__ __forceinline__ double step2(double a, double b, bool hi)
{
    return (hi ? b : a) + dpp<CTRL>(hi ? a : b);
}
template <int CTRL> __device__ __forceinline__ float max_dpp(float x)
{
    return fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(x), CTRL, 0xf,
                                                                0xf, false)));
}
/* The sums over 16 lanes of s[0 .. N), and the largest of them as floats, in
   every lane: row_ror 8, row_half_mirror (7 - l in 8 lanes), then quad_perm [2, 3,
   0, 1] and [1, 0, 3, 2] */
template <uint32_t N> __device__ __forceinline__ float largest16(const double *s, uint32_t c)
{
    double x;
    if constexpr (N == 4)
        x = step2<0x141>(step2<0x128>(s[0], s[1], c & 8), step2<0x128>(s[2], s[3], c & 8), c & 4);
    else if constexpr (N == 2)
        x = step<0x141>(step2<0x128>(s[0], s[1], c & 8));
    else
        x = step<0x141>(step<0x128>(s[0]));
    float y = (float)step<0xB1>(step<0x4E>(x));
    if constexpr (N >= 2)
        y = max_dpp<0x128>(y);
    if constexpr (N == 4)
        y = max_dpp<0x141>(y);
    return y;
}

constexpr uint32_t kScoreRows = 16;    /* rows of 16 lanes a workgroup */
/* rows of lanes that share a block where each takes `ht` of `heads` heads: 1, 2
   or 4 */
constexpr uint32_t score_share(uint32_t heads, uint32_t ht)
{
    return heads <= ht ? 1 : heads <= 2 * ht ? 2 : 4;
}

/*
 * A block's 16 lanes take 8 dimensions of every 128 each; HC: 128s of the head
 * size. The query of 4 / HC heads stays in registers, as doubles and as the mask
 * of its positive numbers, while the lanes go from block to block, the next
 * block's bounds asked for before this one's are used (their pages 16 blocks at
 * a time: a load less to wait for at each): a number and head are a
 * bit select, a conversion and a multiply-add. A larger group's heads go to up to
 * four rows of lanes of one wave, which take a block together (bounds and selection
 * of 16 / 2 heads of 256 over 5 x 375 blocks 20.9 -> 18.1 us against one row that
 * goes over the blocks again, 32 / 1 of 128 over 4 x 940 with the attention 34.2 ->
 * 28.6); what is above 16 / HC heads then goes over them again. Bound by those
 * steps where blocks are many: 8673 blocks of 8 KV heads of 128 in 13.5 us, 2.6 TB/s,
 * of which vector instructions 9.5.
 */
template <int HC, uint32_t SHARE>
__global__ __launch_bounds__(256) void score_kernel(const SelectArgs A)
{
    constexpr uint32_t HT = 4 / HC;
    const uint32_t tid = threadIdx.x, si = blockIdx.z, kvh = blockIdx.y;
    const SeqView sv = seq_view(A, si);
    const Blocks bl = blocks_in_sight(A, sv);
    if (bl.n <= A.n_sel)
        return; /* all of them */
    const uint32_t c = tid % 16, hs = tid / 16 % SHARE, hd = A.hd;
    const uint32_t blocks = kScoreRows / SHARE, step = gridDim.x * blocks;
    const uint32_t j0 = blockIdx.x * blocks + tid / 16 / SHARE;
    if (j0 >= bl.n)
        return; /* (a block's rows of 16 lanes are all there or none) */
    const uint32_t *const table = A.table + (size_t)si * A.max_pages + bl.b0;
    float *const out = A.score + ((size_t)si * A.n_kv + kvh) * A.max_pages;
    bool in[HC];
#pragma unroll
    for (int i = 0; i < HC; i++)
        in[i] = 128 * i + 8 * c < hd;
    /* the pages of the next 16 blocks that these lanes come to, one a lane */
    uint32_t pids = 0;
    auto fetch = [&](uint32_t j) {
        const uint64_t mine = j + (uint64_t)c * step;
        pids = table[mine < bl.n ? mine : bl.n - 1];
        pids = pids < A.n_pages ? pids : 0;
    };
    auto boxes = [&](uint32_t k, h8 *lo, h8 *hi) {
        const uint32_t pid = __shfl(pids, (int)((tid & 48) + k % 16), 64);
        const _Float16 *const box = A.bounds + ((size_t)pid * A.n_kv + kvh) * 2 * hd;
#pragma unroll
        for (int i = 0; i < HC; i++) {
            const uint32_t d = in[i] ? 128 * i + 8 * c : 0;
            lo[i] = *(const h8 *)(box + d);
            hi[i] = *(const h8 *)(box + hd + d);
        }
    };
    fetch(j0);
    /* (a row of lanes past the group's heads takes the first ones again: the largest
       stays what it is) */
    for (uint32_t p0 = 0; p0 < A.group; p0 += HT * SHARE) {
        const uint32_t mine = p0 + HT * hs, h0 = mine < A.group ? mine : p0;
        const float *const q =
            A.q + (size_t)sv.row * A.q_stride + ((size_t)kvh * A.group + h0) * hd;
        double x[HT][HC][8];
        uint32_t m[HT][HC][8];
#pragma unroll
        for (uint32_t h = 0; h < HT; h++)
#pragma unroll
            for (int i = 0; i < HC; i++) {
                const bool ok = in[i] && h0 + h < A.group;
                const float *const p = q + (ok ? (size_t)h * hd + 128 * i + 8 * c : 0);
                const f4 a = *(const f4 *)p, b = *(const f4 *)(p + 4);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float y = e < 4 ? a[e & 3] : b[e & 3];
                    y = !ok ? 0.0f : A.negate ? -y : y;
                    x[h][i][e] = (double)y;
                    m[h][i][e] = y > 0.0f ? 0xFFFFFFFFu : 0;
                }
            }
        h8 lo[HC], hi[HC];
        if (p0 && (bl.n - 1 - j0) / step >= 16)
            fetch(j0);
        boxes(0, lo, hi);
        for (uint32_t j = j0, k = 1; j < bl.n; j += step, k++) {
            uint32_t l[HC][8], u[HC][8];
#pragma unroll
            for (int i = 0; i < HC; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    l[i][e] = __float_as_uint((float)lo[i][e]);
                    u[i][e] = __float_as_uint((float)hi[i][e]);
                }
            if (j + step < bl.n) {
                if (k % 16 == 0)
                    fetch(j + step);
                boxes(k, lo, hi);
            }
            double sum[HT];
#pragma unroll
            for (uint32_t h = 0; h < HT; h++) {
                double s = 0.0;
#pragma unroll
                for (int i = 0; i < HC; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const uint32_t k = m[h][i][e];
                        const float b = __uint_as_float((u[i][e] & k) | (l[i][e] & ~k));
                        s = __builtin_fma(x[h][i][e], (double)b, s);
                    }
                /* (a head past the group: the first one again) */
                sum[h] = h0 + h < A.group ? s : sum[0];
            }
            float best = largest16<HT>(sum, c);
            if constexpr (SHARE > 1)
                best = fmaxf(best, __shfl_xor(best, 16, 64));
            if constexpr (SHARE > 2)
                best = fmaxf(best, __shfl_xor(best, 32, 64));
            if (c == 0 && hs == 0)
                out[j] = p0 == 0 ? best : fmaxf(best, out[j]);
        }
    }
}

constexpr uint32_t kPickThreads = 512;
constexpr uint32_t kPickWaves = kPickThreads / 64;
constexpr uint32_t kPickKeys = 8;      /* keys a thread keeps in registers */

/* a score's place in order, as a whole number */
__device__ __forceinline__ uint32_t score_key(float x)
{
    const uint32_t u = __float_as_uint(x + 0.0f); /* (-0 is 0) */
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

/* the largest over the wave, in lane 63 */
__device__ __forceinline__ uint32_t max_wave(uint32_t x)
{
    auto up = [&](uint32_t y) { x = y > x ? y : x; };
    up(shifted<0x111, 0xf>(x));
    up(shifted<0x112, 0xf>(x));
    up(shifted<0x114, 0xf>(x));
    up(shifted<0x118, 0xf>(x));
    up(shifted<0x142, 0xa>(x));
    up(shifted<0x143, 0xc>(x));
    return x;
}

/*
 * One workgroup a (sequence, KV head). Of the blocks that are not forced, the
 * `want`-th largest key is found 8 bits at a time, from the highest bit in which
 * they differ at all, by a histogram of the keys that share the bits found so
 * far; it is enough to know the bits above which exactly `want` keys lie. Then
 * each thread counts its own chosen blocks - neighbours, so that a scan of the
 * counts puts them in order - and writes them. REG: the thread's keys stay in
 * registers; else they are read again at each step. Bound by its chain of steps:
 * 512 threads measured best (2000 blocks, with bounds, scores and the attention: 25.6
 * us, with 256 threads 26.5, with 1024 26.0; this kernel alone 6.3 under the tracer).
 */
template <bool REG> __device__ void pick(const SelectArgs &A, const Blocks &bl, const float *score,
                                         uint32_t *sel)
{
    __shared__ __attribute__((aligned(16))) uint32_t sHist[4][256];
    __shared__ uint32_t sHigh[kPickWaves], sUnder[kPickWaves];
    __shared__ uint32_t sAbove[kPickWaves], sAt[kPickWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t per = (bl.n + kPickThreads - 1) / kPickThreads, first = tid * per;
    const uint32_t mine = first >= bl.n ? 0 : bl.n - first < per ? bl.n - first : per;
    auto forced = [&](uint32_t j) { return j < A.first || j >= bl.n - A.last; };
    uint32_t kept[REG ? kPickKeys : 1];
    if constexpr (REG) {
#pragma unroll
        for (uint32_t r = 0; r < kPickKeys; r++)
            if (r < mine)
                kept[r] = score_key(score[first + r]);
    }
    /* f(j, key) for the thread's blocks that are not forced */
    auto each = [&](auto f) {
        if constexpr (REG) {
#pragma unroll
            for (uint32_t r = 0; r < kPickKeys; r++)
                if (r < mine && !forced(first + r))
                    f(first + r, kept[r]);
        } else {
            for (uint32_t r = 0; r < mine; r++)
                if (!forced(first + r))
                    f(first + r, score_key(score[first + r]));
        }
    };
    /* the largest key, and of the keys' complements (for the smallest) */
    uint32_t high = 0, under = 0;
    each([&](uint32_t, uint32_t k) {
        high = k > high ? k : high;
        under = ~k > under ? ~k : under;
    });
    high = max_wave(high);
    under = max_wave(under);
    if (lane == 63) {
        sHigh[w] = high;
        sUnder[w] = under;
    }
    for (uint32_t i = tid; i < 1024; i += kPickThreads)
        ((uint32_t *)sHist)[i] = 0;
    __syncthreads();
    high = under = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPickWaves; i++) {
        high = sHigh[i] > high ? sHigh[i] : high;
        under = sUnder[i] > under ? sUnder[i] : under;
    }
    high = __builtin_amdgcn_readfirstlane(high);
    const uint32_t differ = high ^ ~__builtin_amdgcn_readfirstlane(under);
    /* keys >= edge with the bits of `mask` are chosen, those equal to it in them
       until `want` is used up */
    uint32_t want = A.n_sel - A.first - A.last, bits = differ ? 32 - __builtin_clz(differ) : 0;
    uint32_t mask = bits == 32 ? 0 : 0xFFFFFFFFu << bits, edge = high & mask;
    for (int pass = 0; bits > 0 && want > 0; pass++) {
        const uint32_t shift = bits > 8 ? bits - 8 : 0, digits = (1u << (bits - shift)) - 1;
        each([&](uint32_t, uint32_t k) {
            if ((k & mask) == edge)
                atomicAdd(&sHist[pass][k >> shift & digits], 1u);
        });
        __syncthreads();
        /* the bin of the want-th from the top, in every wave: 4 bins a lane from the
           top one down */
        const u4 n = *(const u4 *)&sHist[pass][252 - 4 * lane];
        const uint32_t b1 = n[3], b2 = b1 + n[2], b3 = b2 + n[1], b4 = b3 + n[0];
        const uint32_t upto = scan_wave(b4), left = want - (upto - b4);
        const uint64_t hit = __ballot(want <= upto);
        const uint32_t e = left <= b1 ? 0 : left <= b2 ? 1 : left <= b3 ? 2 : 3;
        const uint32_t over = e == 0 ? 0 : e == 1 ? b1 : e == 2 ? b2 : b3;
        const uint32_t l = (uint32_t)__builtin_ctzll(hit);
        const uint32_t digit = __builtin_amdgcn_readlane(255 - (4 * lane + e), l);
        const uint32_t in = __builtin_amdgcn_readlane(n[3 - e], l);
        want = __builtin_amdgcn_readlane(left - over, l);
        bits = shift;
        mask |= digits << shift;
        edge |= digit << shift;
        if (want == in)
            break; /* all of that bin */
    }
    uint32_t above = 0, at = 0;
    each([&](uint32_t, uint32_t k) {
        above += (k & mask) > edge;
        at += (k & mask) == edge;
    });
    /* (the forced ones count as above) */
    for (uint32_t r = 0; r < mine; r++)
        above += forced(first + r);
    const uint32_t sa = scan_wave(above), st = scan_wave(at);
    if (lane == 63) {
        sAbove[w] = sa;
        sAt[w] = st;
    }
    __syncthreads();
    uint32_t na = sa - above, nt = st - at;
    for (uint32_t i = 0; i < kPickWaves; i++) {
        na += i < w ? sAbove[i] : 0;
        nt += i < w ? sAt[i] : 0;
    }
    auto put = [&](uint32_t j, bool over, bool equal) {
        if (over || (equal && nt < want))
            sel[na + (nt < want ? nt : want)] = bl.b0 + j;
        na += over;
        nt += equal;
    };
    if constexpr (REG) {
#pragma unroll
        for (uint32_t r = 0; r < kPickKeys; r++)
            if (r < mine) {
                const bool f = forced(first + r);
                put(first + r, f || (kept[r] & mask) > edge, !f && (kept[r] & mask) == edge);
            }
    } else {
        for (uint32_t r = 0; r < mine; r++) {
            const bool f = forced(first + r);
            const uint32_t k = f ? 0 : score_key(score[first + r]) & mask;
            put(first + r, f || k > edge, !f && k == edge);
        }
    }
}

__global__ __launch_bounds__(kPickThreads) void pick_kernel(const SelectArgs A)
{
    const uint32_t tid = threadIdx.x;
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
    if (bl.n <= kPickKeys * kPickThreads)
        pick<true>(A, bl, score, sel);
    else
        pick<false>(A, bl, score, sel);
}

}  // namespace

hipError_t launch_bounds(const BoundsArgs &a, hipStream_t s)
{
    const dim3 grid(a.max_blocks * bound_slices(a.hd), a.n_kv, a.n_seqs);
    if (a.kv == kI8)
        hipLaunchKernelGGL(bounds_kernel<kI8>, grid, dim3(256), 0, s, a);
    else if (a.kv == kI16)
        hipLaunchKernelGGL(bounds_kernel<kI16>, grid, dim3(256), 0, s, a);
    else if (a.kv == kF16)
        hipLaunchKernelGGL(bounds_kernel<kF16>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(bounds_kernel<kF32>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int HC>
static void launch_scores(const SelectArgs &a, uint32_t share, dim3 grid, hipStream_t s)
{
    if (share == 1)
        hipLaunchKernelGGL((score_kernel<HC, 1>), grid, dim3(256), 0, s, a);
    else if (share == 2)
        hipLaunchKernelGGL((score_kernel<HC, 2>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((score_kernel<HC, 4>), grid, dim3(256), 0, s, a);
}

hipError_t launch_select(const SelectArgs &a, hipStream_t s)
{
    /* as many workgroups as hold the table's blocks once, no more than fill the
       device (max_pages may be far above the lengths, and each workgroup makes
       its query first) */
    const uint32_t pairs = a.n_seqs * a.n_kv;
    const uint32_t ht = a.hd <= 128 ? 4 : a.hd <= 256 ? 2 : 1;
    const uint32_t share = score_share(a.group, ht), blocks = kScoreRows / share;
    uint32_t x = (a.max_pages + blocks - 1) / blocks;
    const uint32_t most = pairs < 4 * a.cus ? 4 * a.cus / pairs : 1;
    x = x < most ? x : most;
    const dim3 grid(x, a.n_kv, a.n_seqs);
    if (a.hd <= 128)
        launch_scores<1>(a, share, grid, s);
    else if (a.hd <= 256)
        launch_scores<2>(a, share, grid, s);
    else
        launch_scores<4>(a, share, grid, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return e;
    hipLaunchKernelGGL(pick_kernel, dim3(pairs), dim3(kPickThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace janas
