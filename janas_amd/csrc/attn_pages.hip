/*
 * attn_pages.hip - attention of one new token of every sequence over a paged
 * cache, for CDNA4 (gfx950).
 *
 *   o = sum_p w_p v_p / sum_p w_p,  w_p = 2^(x_p - m),  x_p = log2(e) scale q.k_p
 *
 * over the positions in sight, or those of a KV head's selected blocks.
 *
 *   pages_kernel   one workgroup (4 waves) per (sequence, KV head, tile of
 *                  query rows, split of the positions). A wave walks its own
 *                  positions in units of 16 - a page holds whole units - with
 *                  one running softmax; nothing is shared until the four waves
 *                  are joined at the end.
 *   pages_merge_kernel  joins a row's splits, in order, and applies the gate.
 *
 * Both find their work on the device from the sequences' lengths (plan_splits),
 * so a launch depends on none and can be captured.
 *
 * Operands go from memory to registers in the shape the matrix cores take
 * them, without LDS. Scores, S^T = K Q^T, contract over the head dimension in
 * any order: a lane's 16 bytes of one row are A operands as they are. The value
 * product contracts over positions: a lane of 16 takes the same 8 columns of
 * four rows, and byte permutes pair the rows' numbers, one a register. So
 * output column 8 n + e of a unit of 128 sits in lane n of product e.
 *
 * Precision as in attn_split.hip: query and weights as two f16 planes (query
 * row r in MFMA columns 2 r, 2 r + 1), cached integers and halves exact, f32
 * sums. An f32 cache takes f32 products (v_mfma_f32_16x16x4_f32) instead, 16
 * query rows a workgroup.
 */
#include <math.h>
#include <stdint.h>

#include <hip/hip_runtime.h>

#include "attn_elem.h"
#include "attn_pages.h"

#pragma clang fp contract(off)

namespace janas {
namespace {

constexpr int kPW = 4;          /* waves a workgroup */
constexpr uint32_t kUnit = 16;  /* positions a unit */
/* A row's reference score is renewed only once a score passes it by 2^8: the
   weights then stay below 2^8, and their planes are taken of 2^7 times them, so
   f16's smallest step is 2^-31 of a weight of 1 */
constexpr float kLazy = 8.0f;
constexpr int kUp = 7;

/* ---- which positions a workgroup takes ------------------------------------ */

/* a sequence's units of 16 positions (0: no part, nothing in sight, or bad) */
template <bool SEL>
__device__ __forceinline__ uint32_t seq_units(const PagesArgs &A, const SeqView &s)
{
    if (!s.part || s.bad || s.end <= s.lo)
        return 0;
    if constexpr (SEL) {
        const uint32_t nb = (s.end + (1u << A.page_log) - 1) >> A.page_log;
        return (nb < A.n_sel ? nb : A.n_sel) << (A.page_log - 4);
    } else {
        return (s.end + kUnit - 1) / kUnit - s.lo / kUnit;
    }
}

__device__ __forceinline__ uint32_t sum_wave(uint32_t x)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        x += __shfl_xor(x, o, 64);
    return x;
}
/* sum over the lanes up to and with this one */
__device__ __forceinline__ uint32_t scan_wave(uint32_t x, uint32_t lane)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(x, o, 64);
        x += lane >= (uint32_t)o ? y : 0;
    }
    return x;
}

/* units a split takes at least: 4 a wave. Below that a wave's start (length,
   table, query, first rows: a chain of reads) is most of its time. */
constexpr uint32_t kLeastUnits = 4 * kPW;

/* The units a split aims at: all sequences' units over the splits that a KV
   head's row tile has (A.share). Every wave finds it for itself, a lane a
   sequence. */
template <bool SEL>
__device__ __forceinline__ uint32_t split_units(const PagesArgs &A, uint32_t lane)
{
    uint64_t total = 0;
    for (uint32_t i0 = 0; i0 < A.n_seqs; i0 += 64) {
        const uint32_t i = i0 + lane;
        /* below 2^27 a lane (2^31 positions): 64 of them need a bit more */
        const uint32_t u = i < A.n_seqs ? seq_units<SEL>(A, seq_view(A, i)) : 0;
        total += (uint64_t)sum_wave(u >> 16) * 65536 + sum_wave(u & 0xFFFF);
    }
    const uint64_t per = (total + A.share - 1) / A.share;
    return per < kLeastUnits ? kLeastUnits : per < 0xFFFFFFFFu ? (uint32_t)per : 0xFFFFFFFFu;
}

struct Split {
    uint32_t seq, index, count, units; /* split `index` of `count`, of units */
};

/* split number `at` of the call (per KV head and row tile), or the splits
   before sequence `want` (index) and its own (count) */
template <bool SEL>
__device__ __forceinline__ Split find_split(const PagesArgs &A, uint32_t lane, uint32_t at,
                                            uint32_t want)
{
    Split f{kNone, 0, 0, 0};
    const uint32_t per = split_units<SEL>(A, lane);
    uint32_t before = 0;
    for (uint32_t i0 = 0; i0 < A.n_seqs; i0 += 64) {
        const uint32_t i = i0 + lane;
        const uint32_t u = i < A.n_seqs ? seq_units<SEL>(A, seq_view(A, i)) : 0;
        const uint32_t n = u ? (u - 1) / per + 1 : 0;
        const uint32_t end = scan_wave(n, lane) + before;
        const uint64_t past = want == kNone ? __ballot(end > at) : __ballot(i == want);
        if (past) {
            const uint32_t l = (uint32_t)__builtin_ctzll(past);
            f.seq = i0 + l;
            f.count = __builtin_amdgcn_readlane(n, l);
            f.units = __builtin_amdgcn_readlane(u, l);
            const uint32_t first = __builtin_amdgcn_readlane(end, l) - f.count;
            f.index = want == kNone ? at - first : first;
            return f;
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    return f;
}

/* ---- raw words of a row ------------------------------------------------------ */

template <int W> struct Words;
template <> struct Words<1> { typedef uint32_t T; };
template <> struct Words<2> { typedef uint32_t T __attribute__((ext_vector_type(2))); };
template <> struct Words<4> { typedef u4 T; };
template <int W> __device__ __forceinline__ uint32_t word(const typename Words<W>::T &x, int i)
{
    if constexpr (W == 1)
        return x;
    else
        return x[i];
}

template <int T, int D> struct PS {
    static constexpr int EB = Elem<T>::bytes;
    static constexpr bool F32 = T == kF32;
    static constexpr bool SCALED = T == kI8 || T == kI16;
    static constexpr int ROWS = F32 ? 16 : 8;        /* query rows a workgroup */
    static constexpr int KL = D * EB / 64;           /* 16-byte loads of a K row a lane */
    static constexpr int VN = F32 || D == 64 ? 4 : 8; /* columns a V load */
    static constexpr int VU = D / (16 * VN);         /* V loads of a row a lane */
    static constexpr int VW = VN * EB / 4;           /* words of one */
    static constexpr int NT = D / 16;                /* column tiles */
    static constexpr int DP = Elem<T>::planes;
};

/* numbers e of four rows' V words as B operands, one a plane */
template <int T, int VW>
__device__ __forceinline__ void value_operand(const typename Words<VW>::T *v, int e, h4 *b)
{
    uint32_t p[2], q[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if constexpr (T == kF16) {
            p[h] = __builtin_amdgcn_perm(word<VW>(v[2 * h + 1], e / 2), word<VW>(v[2 * h], e / 2),
                                         e & 1 ? 0x07060302u : 0x05040100u);
        } else if constexpr (T == kI8) {
            /* b ^ 0x80 under the exponent byte 0x64 is the half 1152 + b */
            const uint32_t c = e & 3;
            const uint32_t x = __builtin_amdgcn_perm(
                word<VW>(v[2 * h + 1], e / 4), word<VW>(v[2 * h], e / 4),
                0x0c000c00u | (4 + c) << 16 | c);
            const h2 y = __builtin_bit_cast(h2, x ^ 0x64806480u) -
                         h2{(_Float16)1152.0f, (_Float16)1152.0f};
            p[h] = __builtin_bit_cast(uint32_t, y);
        } else {
            /* 256 (x >> 8) and x & 255 */
            const uint32_t c = 2 * (e & 1);
            const uint32_t a = word<VW>(v[2 * h + 1], e / 2), d = word<VW>(v[2 * h], e / 2);
            const uint32_t lo = __builtin_amdgcn_perm(a, d, 0x0c000c00u | (4 + c) << 16 | c);
            const uint32_t hi = __builtin_amdgcn_perm(a, d, 0x0c000c00u | (5 + c) << 16 | (1 + c));
            const h2 y = __builtin_bit_cast(h2, lo | 0x64006400u) -
                         h2{(_Float16)1024.0f, (_Float16)1024.0f};
            const h2 z = (__builtin_bit_cast(h2, hi ^ 0x64806480u) -
                          h2{(_Float16)1152.0f, (_Float16)1152.0f}) *
                         h2{(_Float16)256.0f, (_Float16)256.0f};
            p[h] = __builtin_bit_cast(uint32_t, z);
            q[h] = __builtin_bit_cast(uint32_t, y);
        }
    }
    b[0] = __builtin_bit_cast(h4, make_uint2(p[0], p[1]));
    if constexpr (T == kI16)
        b[1] = __builtin_bit_cast(h4, make_uint2(q[0], q[1]));
}

__device__ __forceinline__ float sigmoid(float g) { return 1.0f / (1.0f + expf(-g)); }

/* the exponent field of a non-negative number */
__device__ __forceinline__ uint32_t exponent(float x) { return (__float_as_uint(x) >> 23) & 255; }

/* ---- the kernel ---------------------------------------------------------------- */

template <int T, int D, bool SEL>
__global__ __launch_bounds__(kPW * 64) void pages_kernel(const PagesArgs A)
{
    using S = PS<T, D>;
    constexpr int EB = S::EB, KL = S::KL, VN = S::VN, VU = S::VU, VW = S::VW, NT = S::NT;
    constexpr int DP = S::DP, ROWS = S::ROWS;
    constexpr bool F32 = S::F32, SCALED = S::SCALED;
    typedef typename Words<VW>::T VT;
    __shared__ __attribute__((aligned(16))) float sO[kPW][ROWS][D];
    __shared__ float sM[kPW][ROWS], sL[kPW][ROWS];
    __shared__ float sE[kPW];

    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t g = lane >> 4, n = lane & 15;
    const uint32_t tiles = A.n_kv * A.rtiles, tile = blockIdx.x % tiles;
    const Split sp = find_split<SEL>(A, lane, blockIdx.x / tiles, kNone);
    if (sp.seq == kNone)
        return;
    const SeqView sv = seq_view(A, sp.seq);
    const uint32_t hd = A.hd, G = A.group, rowb = hd * EB;
    const uint32_t kvh = tile / A.rtiles, r0 = tile % A.rtiles * ROWS;
    const uint32_t rows = G - r0 < ROWS ? G - r0 : ROWS;
    const uint32_t page = 1u << A.page_log, upp = page / kUnit, upp_log = A.page_log - 4;

    /* the split's units, and the wave's quarter of them */
    const uint32_t ua = (uint32_t)((uint64_t)sp.units * sp.index / sp.count);
    const uint32_t ub = (uint32_t)((uint64_t)sp.units * (sp.index + 1) / sp.count);
    const uint32_t wa = ua + (ub - ua) * w / kPW, wb = ua + (ub - ua) * (w + 1) / kPW;
    /* units counted from the first page of the list */
    const uint32_t u0 = SEL ? 0 : sv.lo / kUnit;
    const uint32_t first = wa + u0, last = wb + u0; /* [first, last) */

    /* ---- pages: lane i holds entry e0 + i of the wave's list - the block's page
       and its number ---- */
    const uint32_t nb = (sv.end + page - 1) >> A.page_log;
    const uint32_t *const trow = A.table + (size_t)sp.seq * A.max_pages;
    const uint32_t *const srow = SEL ? A.sel + ((size_t)sp.seq * A.n_kv + kvh) * A.n_sel : nullptr;
    uint32_t e0 = first >> upp_log, pid = 0, blk = 0;
    bool bad = false;
    auto fetch = [&](uint32_t from) {
        const uint32_t e = from + lane;
        const bool mine = e <= (last - 1) >> upp_log;
        blk = mine ? e : kNone;
        if constexpr (SEL) {
            if (mine)
                blk = srow[e];
        }
        pid = 0;
        if (blk < nb) {
            pid = trow[blk];
            bad |= pid >= A.n_pages;
            pid = pid < A.n_pages ? pid : 0;
        } else {
            blk = kNone;
        }
    };

    /* a unit: its page and KV head's rows, its first row and position (past
       the end: none of it is in sight) */
    struct Unit {
        size_t row;
        uint32_t pos;
    };
    auto unit_of = [&](uint32_t u) {
        const uint32_t e = u >> upp_log;
        if (e - e0 >= 64) {
            e0 = e;
            fetch(e0);
        }
        const uint32_t p = __builtin_amdgcn_readlane(pid, e - e0);
        const uint32_t b = __builtin_amdgcn_readlane(blk, e - e0);
        const uint32_t in = (u & (upp - 1)) * kUnit;
        Unit x;
        x.row = (((size_t)p * A.n_kv + kvh) << A.page_log) + in;
        x.pos = b == kNone ? kNone - kUnit : (b << A.page_log) + in;
        return x;
    };

    u4 kr[KL];
    VT vr[4][VU];
    f4 ks{1, 1, 1, 1}, vs{1, 1, 1, 1};
    /* the lane's bytes of a K row, and its columns of a V row */
    uint32_t kat[KL], vat[VU];
    bool kback[KL];
#pragma unroll
    for (int i = 0; i < KL; i++) {
        const uint32_t cb = 64 * i + 16 * g;
        kback[i] = false;
        if constexpr (EB == 1)
            kat[i] = unit_at(cb, rowb, kback[i]);
        else
            kat[i] = cb < rowb ? cb : 0;
        kat[i] += n * rowb;
    }
#pragma unroll
    for (int u = 0; u < VU; u++) {
        const uint32_t c = 16 * VN * u + VN * n;
        vat[u] = (c < hd ? c : 0) * EB;
    }
    auto load_k = [&](const Unit &x) {
        const char *const p = (const char *)A.k + x.row * rowb;
#pragma unroll
        for (int i = 0; i < KL; i++)
            kr[i] = __builtin_nontemporal_load((const u4 *)(p + kat[i]));
        if constexpr (SCALED)
            ks = *(const f4 *)(A.ks + x.row + 4 * g);
    };
    /* value rows past the sequence's are read as its last one (they weigh 0,
       but what is there may be no number) */
    auto load_v = [&](const Unit &x) {
        const uint32_t hi = x.pos < sv.end ? (sv.end - 1 - x.pos < 15 ? sv.end - 1 - x.pos : 15) : 0;
        const uint32_t lo = x.pos < sv.lo ? (sv.lo - x.pos < 15 ? sv.lo - x.pos : 15) : 0;
        const char *const p = (const char *)A.v + x.row * rowb;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t r = 4 * g + j;
            r = r > lo ? r : lo;
            r = r < hi ? r : hi;
#pragma unroll
            for (int u = 0; u < VU; u++)
                vr[j][u] = __builtin_nontemporal_load((const VT *)(p + r * rowb + vat[u]));
        }
        if constexpr (SCALED)
            vs = *(const f4 *)(A.vs + x.row + 4 * g);
    };

    /* ---- the query: row n / 2 (f32: n) as the B operand of each K load ---- */
    constexpr int QN = 16 / EB;      /* numbers of a K load: 16, 8 or 4 */
    h8 qb[F32 ? 1 : KL][F32 ? 1 : QN / 8];
    f4 qf[F32 ? KL : 1];
    float qs2;
    {
        const uint32_t qr = F32 ? n : n >> 1;
        const bool ok = qr < rows;
        const float *const src =
            A.q + (size_t)sv.row * A.q_stride + (size_t)(kvh * G + r0 + (ok ? qr : 0)) * hd;
        f4 x[KL][QN / 4];
        float mx = 0.0f;
#pragma unroll
        for (int i = 0; i < KL; i++)
#pragma unroll
            for (int j = 0; j < QN / 4; j++) {
                const uint32_t c = QN * (4 * i + g) + 4 * j;
                x[i][j] = *(const f4 *)(src + (c < hd ? c : 0));
                if (!ok || c >= hd)
                    x[i][j] = f4{0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; e++)
                    mx = fmaxf(mx, fabsf(x[i][j][e]));
            }
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < KL; i++)
                qf[i] = x[i][0];
            qs2 = A.scale * kLog2e;
        } else {
            /* scaled by 2^ex so that the row's largest lies in [2^13, 2^14);
               even columns take the high plane, odd ones what is left */
            mx = max_x32(max_x16(mx));
            int ex = 0;
            if (mx > 0.0f && mx < INFINITY) {
                frexpf(mx, &ex);
                ex = 14 - ex;
            }
            const float up = ldexpf(1.0f, ex);
#pragma unroll
            for (int i = 0; i < KL; i++)
#pragma unroll
                for (int j = 0; j < QN / 4; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        _Float16 hi, lo;
                        split_hl(x[i][j][e] * up, hi, lo);
                        qb[i][j / 2][4 * (j & 1) + e] = n & 1 ? lo : hi;
                    }
            qs2 = ldexpf(1.0f, -ex) * A.scale * kLog2e;
        }
    }

    /* ---- the wave's positions ---- */
    f4 o[NT];
#pragma unroll
    for (int t = 0; t < NT; t++)
        o[t] = f4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;  /* of the lane's row; l its own positions' */
    uint32_t ev = 64;               /* exponent field that the value scales stay
                                       within */
    float vup = 0.0f;               /* a weight's factor: 2^kUp over theirs */
    const float keep = lane & 1 ? -1.0f : -0.0f;
    if (first < last) {
        fetch(e0);
        Unit x = unit_of(first);
        load_k(x);
        load_v(x);
        for (uint32_t u = first; u < last; u++) {
            const Unit now = x;
            const bool more = u + 1 < last;
            if (more)
                x = unit_of(u + 1);
            /* scores: lane holds positions 4 g + j of MFMA column n */
            f4 s{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KL; i++) {
                if constexpr (F32) {
                    const f4 kf = __builtin_bit_cast(f4, kr[i]);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[i][e], s, 0, 0, 0);
                } else if constexpr (T == kI8) {
                    const u4 y = unit_fix(kr[i], kback[i]);
                    s = mfma(i8_widen8(y.x, y.y), qb[i][0], s);
                    s = mfma(i8_widen8(y.z, y.w), qb[i][1], s);
                } else if constexpr (T == kI16) {
                    h8 hi, lo;
                    i16_planes8(kr[i].x, kr[i].y, kr[i].z, kr[i].w, hi, lo);
                    s = mfma(hi, qb[i][0], s);
                    s = mfma(lo, qb[i][0], s);
                } else {
                    s = mfma(__builtin_bit_cast(h8, kr[i]), qb[i][0], s);
                }
            }
            const f4 kz = ks;
            if (more)
                load_k(x);
            if (now.pos < sv.end && now.pos + kUnit > sv.lo) {
                f4 vz = vs;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (!F32)
                        s[j] += from_x1(s[j]);
                    s[j] *= qs2;
                    if constexpr (SCALED)
                        s[j] *= kz[j];
                }
                if (now.pos < sv.lo || now.pos + kUnit > sv.end) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t p = now.pos + 4 * g + j;
                        const bool in = p >= sv.lo && p < sv.end;
                        s[j] = in ? s[j] : -INFINITY;
                        vz[j] = in ? vz[j] : 0.0f;
                    }
                }
                const float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
                uint32_t ex = 0;
                if constexpr (SCALED)
                    ex = exponent(fmaxf(fmaxf(vz[0], vz[1]), fmaxf(vz[2], vz[3])));
                if (__any(top > m + kLazy || ex > ev)) {
                    /* new references; what is summed so far follows */
                    const float mn = fmaxf(m, max_x32(max_x16(top)));
                    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
                    l *= f;
                    float fe = 1.0f;
                    if constexpr (SCALED) {
                        const uint32_t en = (uint32_t)fmaxf((float)ev, max_x32(max_x16((float)ex)));
                        fe = ldexpf(1.0f, (int)ev - (int)en);
                        ev = en;
                    }
                    vup = ldexpf(1.0f, kUp + (SCALED ? 126 - (int)ev : 0));
                    float fr[4];
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        fr[i] = __shfl(f, (int)(4 * g + (F32 ? i : i & 2)), 64) * fe;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            o[t][i] *= fr[i];
                }
                const float mm = m == -INFINITY ? 0.0f : m;
                h4 pa;
                f4 pf;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float p = __builtin_amdgcn_exp2f(s[j] - mm);
                    l += p;
                    pf[j] = p;
                    if constexpr (!F32) {
                        float pv = p * vup;
                        if constexpr (SCALED)
                            pv *= vz[j];
                        asm volatile("" : "+v"(pv));
                        const float hi = (float)(_Float16)pv;
                        pa[j] = (_Float16)__builtin_fmaf(keep, hi, pv);
                    }
                }
                /* values: product e of a unit of columns */
#pragma unroll
                for (int c = 0; c < VU; c++)
#pragma unroll
                    for (int e = 0; e < VN; e++) {
                        const int t = c * VN + e;
                        if constexpr (F32) {
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    pf[j], __uint_as_float(word<VW>(vr[j][c], e)), o[t], 0, 0, 0);
                        } else {
                            const VT v4[4] = {vr[0][c], vr[1][c], vr[2][c], vr[3][c]};
                            h4 vb[DP];
                            value_operand<T, VW>(v4, e, vb);
#pragma unroll
                            for (int d = 0; d < DP; d++)
                                o[t] = __builtin_amdgcn_mfma_f32_16x16x16f16(pa, vb[d], o[t], 0, 0, 0);
                        }
                    }
            }
            if (more)
                load_v(x);
        }
    }

    /* ---- the waves joined ---- */
    l = sum_x32(sum_x16(l));
    if (__any(bad))
        l = NAN;
    if (F32 ? lane < 16 : lane < 16 && !(lane & 1)) {
        const uint32_t r = F32 ? lane : lane >> 1;
        /* a bad wave may have no score of its own */
        sM[w][r] = l != l && m == -INFINITY ? 0.0f : m;
        sL[w][r] = l;
    }
    if (lane == 0)
        sE[w] = F32 ? 1.0f : ldexpf(1.0f, -kUp - (SCALED ? 126 - (int)ev : 0));
#pragma unroll
    for (int c = 0; c < VU; c++)
#pragma unroll
        for (int i = 0; i < (F32 ? 4 : 2); i++) {
            const uint32_t r = F32 ? 4 * g + i : 2 * g + i;
            if (r >= rows)
                continue;
            float y[VN];
#pragma unroll
            for (int e = 0; e < VN; e++)
                y[e] = F32 ? o[c * VN + e][i] : o[c * VN + e][2 * i] + o[c * VN + e][2 * i + 1];
#pragma unroll
            for (int e = 0; e < VN; e += 4)
                *(f4 *)&sO[w][r][16 * VN * c + VN * n + e] = f4{y[e], y[e + 1], y[e + 2], y[e + 3]};
        }
    __syncthreads();
    const uint32_t c4 = hd / 4;      /* (hd: a multiple of 8) */
    for (uint32_t t = tid; t < rows * c4; t += kPW * 64) {
        const uint32_t r = t / c4, c = 4 * (t % c4);
        const float mx = fmaxf(fmaxf(sM[0][r], sM[1][r]), fmaxf(sM[2][r], sM[3][r]));
        f4 y{0, 0, 0, 0};
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kPW; i++) {
            const float f = sM[i][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sM[i][r] - mx);
            sum += f * sL[i][r];
            const f4 x = *(const f4 *)&sO[i][r][c];
            const float fo = f * sE[i];
#pragma unroll
            for (int e = 0; e < 4; e++)
                y[e] += fo * x[e];
        }
        if (sp.count > 1) {
            const size_t pr = (size_t)blockIdx.x * ROWS + r;
            *(f4 *)(A.part_acc + pr * hd + c) = y;
            if (c == 0)
                *(float2 *)(A.part_ml + 2 * pr) = make_float2(mx, sum);
            continue;
        }
        const size_t hr = (size_t)sv.row * A.n_head + kvh * G + r0 + r;
        /* (nothing in sight, in selected blocks: 0) */
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        f4 sg{1, 1, 1, 1};
        if (A.gate_mode == kGateElem)
            sg = *(const f4 *)(A.gate + hr * hd + c);
        else if (A.gate_mode == kGateHead)
            sg[0] = sg[1] = sg[2] = sg[3] = A.gate[hr];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            y[e] *= inv;
            if (A.gate_mode != kGateNone)
                y[e] *= sigmoid(sg[e]);
        }
        *(f4 *)(A.out + hr * hd + c) = y;
    }
}

/* ---- the merge --------------------------------------------------------------- */

constexpr uint32_t kMCols = 32;              /* columns a workgroup */
constexpr uint32_t kMLanes = kMCols / 4;     /* lanes of a split: a float4 each */
constexpr uint32_t kMGroups = 256 / kMLanes; /* splits at once */
constexpr int kMBatch = 4;

/* A row's splits joined: group i of 32 takes splits i, i + 32, ... with a
   running maximum, the groups of a wave and then the waves are joined in a
   fixed tree. Rows of one split are written by pages_kernel, rows that see
   nothing here: 0, or NaN where the length passes the table. */
template <bool SEL, int ROWS> __global__ __launch_bounds__(256) void pages_merge_kernel(const PagesArgs A)
{
    __shared__ float sM[4], sL[4];
    __shared__ f4 sA[4][kMLanes];
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t hd = A.hd, nd = (hd + kMCols - 1) / kMCols;
    const uint32_t h = blockIdx.x / nd % A.n_head, si = blockIdx.x / nd / A.n_head;
    const uint32_t col = blockIdx.x % nd * kMCols + 4 * (lane % kMLanes);
    const SeqView sv = seq_view(A, si);
    if (!sv.part)
        return;
    const Split sp = find_split<SEL>(A, lane, 0, si);
    if (sp.count == 1)
        return;
    const size_t hr = (size_t)sv.row * A.n_head + h;
    if (sp.count == 0) {
        const float z = sv.bad ? NAN : 0.0f;
        if (tid < kMLanes && col < hd)
            *(f4 *)(A.out + hr * hd + col) = f4{z, z, z, z};
        return;
    }
    const uint32_t kvh = h / A.group, r = h % A.group;
    const uint32_t tiles = A.n_kv * A.rtiles, tile = kvh * A.rtiles + r / ROWS;
    const uint32_t at = col < hd ? col : 0;
    float m = -INFINITY, l = 0.0f;
    f4 a{0, 0, 0, 0};
    for (uint32_t i0 = tid / kMLanes; i0 < sp.count; i0 += kMGroups * kMBatch) {
        float2 ml[kMBatch];
        f4 x[kMBatch];
#pragma unroll
        for (int b = 0; b < kMBatch; b++) {
            uint32_t i = i0 + kMGroups * b;
            i = i < sp.count ? i : sp.count - 1;
            const size_t pr = ((size_t)(sp.index + i) * tiles + tile) * ROWS + r % ROWS;
            ml[b] = *(const float2 *)(A.part_ml + 2 * pr);
            x[b] = *(const f4 *)(A.part_acc + pr * hd + at);
        }
        float mn = m;
#pragma unroll
        for (int b = 0; b < kMBatch; b++)
            mn = fmaxf(mn, ml[b].x);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
        a *= f;
        m = mn;
#pragma unroll
        for (int b = 0; b < kMBatch; b++) {
            const bool in = i0 + kMGroups * b < sp.count && ml[b].x != -INFINITY;
            const float e = in ? __builtin_amdgcn_exp2f(ml[b].x - mn) : 0.0f;
            l += in ? e * ml[b].y : 0.0f;
#pragma unroll
            for (int c = 0; c < 4; c++)
                a[c] = __builtin_fmaf(e, x[b][c], a[c]);
        }
    }
    /* the wave's 8 groups, then the 4 waves */
    float mw = m;
#pragma unroll
    for (int o = 8; o < 64; o <<= 1)
        mw = fmaxf(mw, __shfl_xor(mw, o, 64));
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mw);
    l *= f;
    a *= f;
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) {
        l += __shfl_xor(l, o, 64);
#pragma unroll
        for (int c = 0; c < 4; c++)
            a[c] += __shfl_xor(a[c], o, 64);
    }
    if (lane == 0) {
        sM[w] = mw;
        sL[w] = l;
    }
    if (lane < kMLanes)
        sA[w][lane] = a;
    __syncthreads();
    if (tid >= kMLanes || col >= hd)
        return;
    const float mx = fmaxf(fmaxf(sM[0], sM[1]), fmaxf(sM[2], sM[3]));
    float sum = 0.0f;
    f4 y{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float e = sM[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sM[i] - mx);
        sum += e * sL[i];
        y += e * sA[i][lane];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    f4 sg{1, 1, 1, 1};
    if (A.gate_mode == kGateElem)
        sg = *(const f4 *)(A.gate + hr * hd + col);
    else if (A.gate_mode == kGateHead)
        sg[0] = sg[1] = sg[2] = sg[3] = A.gate[hr];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        y[e] *= inv;
        if (A.gate_mode != kGateNone)
            y[e] *= sigmoid(sg[e]);
    }
    *(f4 *)(A.out + hr * hd + col) = y;
}

template <int T, int D> hipError_t launch_sel(const PagesArgs &a, hipStream_t s)
{
    if (a.sel)
        hipLaunchKernelGGL((pages_kernel<T, D, true>), dim3(a.n_wg), dim3(kPW * 64), 0, s, a);
    else
        hipLaunchKernelGGL((pages_kernel<T, D, false>), dim3(a.n_wg), dim3(kPW * 64), 0, s, a);
    return hipGetLastError();
}

template <int T> hipError_t launch_hd(const PagesArgs &a, hipStream_t s)
{
    if (a.hd <= 64)
        return launch_sel<T, 64>(a, s);
    if (a.hd <= 128)
        return launch_sel<T, 128>(a, s);
    if (a.hd <= 256)
        return launch_sel<T, 256>(a, s);
    if constexpr (T != kF32)
        return launch_sel<T, 512>(a, s);
    return hipErrorInvalidValue;
}

}  // namespace

int pages_supported(int kv, uint32_t hd)
{
    /* an f32 row of 512 would not leave the query and the sums in registers;
       an int8 row is read 16 bytes at a time */
    return kv >= kI8 && kv <= kF32 && hd >= (kv == kI8 ? 16u : 8u) && hd % 8 == 0 &&
           hd <= (kv == kF32 ? 256u : 512u);
}

uint32_t pages_share(uint32_t cus, uint32_t tiles)
{
    const uint32_t fill = 4 * cus;
    return fill / tiles > 1 ? fill / tiles : 1;
}

hipError_t launch_pages(int kv, const PagesArgs &a, hipStream_t s)
{
    switch (kv) {
    case kI8:
        return launch_hd<kI8>(a, s);
    case kI16:
        return launch_hd<kI16>(a, s);
    case kF16:
        return launch_hd<kF16>(a, s);
    case kF32:
        return launch_hd<kF32>(a, s);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_pages_merge(int kv, const PagesArgs &a, hipStream_t s)
{
    const uint32_t n_wg = a.n_seqs * a.n_head * ((a.hd + kMCols - 1) / kMCols);
    const bool f32 = kv == kF32;
    if (a.sel && f32)
        hipLaunchKernelGGL((pages_merge_kernel<true, 16>), dim3(n_wg), dim3(256), 0, s, a);
    else if (a.sel)
        hipLaunchKernelGGL((pages_merge_kernel<true, 8>), dim3(n_wg), dim3(256), 0, s, a);
    else if (f32)
        hipLaunchKernelGGL((pages_merge_kernel<false, 16>), dim3(n_wg), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((pages_merge_kernel<false, 8>), dim3(n_wg), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace janas
