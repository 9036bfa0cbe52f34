/*
 * attn_pages.hip - attention of one new token of every sequence over a paged
 * cache, for CDNA4 (gfx950).
 *
 *   o = sum_p w_p v_p / sum_p w_p,  w_p = 2^(x_p - m),  x_p = log2(e) scale q.k_p
 *
 * over the positions in sight, or those of a KV head's selected blocks.
 *
 *   pages_kernel   one workgroup (4 waves) per (sequence, KV head, tile of
 *                  query rows, run of positions). A wave walks its own positions
 *                  in units of 16 - a page holds whole units - with one running
 *                  softmax; nothing is shared until the four waves are joined
 *                  at the end.
 *   pages_merge_kernel  joins the partials of a row that several workgroups
 *                  took, in order, and applies the gate.
 *
 * The work is dealt on the device from the sequences' lengths (Runs), so a
 * launch depends on none and can be captured.
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
 *
 * Bound by memory where there is much to read - 60 sequences of 4170 positions, 32
 * / 8 / 128 f16, in 160 us, 6.4 TB/s with the merge; 90000 positions of 16 / 2 / 512
 * int16 in 73.5, 5.0 - and where there is little by the chain to the first row (length,
 * table, row), some 4 us, and the two launches: 1000 positions of int8 8.2 us.
 */
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

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
    return __builtin_amdgcn_readlane(scan_wave(x), 63);
}

/* units a workgroup takes at least: one a wave */
constexpr uint32_t kLeastUnits = kPW;

/*
 * The work of a launch: the units of all sequences, one sequence after another,
 * cut into runs of `per` - one a workgroup (of each KV head's row tile), A.share
 * of them at most, which is what the device holds at once. Every workgroup then
 * has the same number of units, whatever the lengths are, and one that crosses
 * from a sequence into the next does one after the other. Where there are runs
 * enough for it, each sequence begins a run of its own instead (its units
 * rounded up to whole runs), so that no workgroup has two.
 *
 * Every wave finds its part for itself, a lane a sequence, 64 at a time; what it
 * will want of them stays in LDS. Up to 64 sequences that is one load; above, three
 * passes over them at most, some 18 us a thousand (one sequence of 1000 positions
 * beside empty ones: 5.2 us up to 64, 7.6 of 256, 18.5 of 1024, 72 of 4096).
 */
struct RunsLds {
    uint32_t row[64], lo[64], end[64], units[64];
    uint32_t from[64], to[64];   /* a sequence's units in the launch's */
};

/* (units count in 32 bits, four times as many too: janas_attn_pages_run refuses
   tables that hold more) */
template <bool SEL> struct Runs {
    uint32_t i0, per, whole;     /* units a run; each sequence in whole runs */
    uint32_t runs;               /* of the launch */

    static __device__ __forceinline__ uint32_t units(const PagesArgs &A, uint32_t i, SeqView &s)
    {
        s = SeqView{};
        if (i >= A.n_seqs)
            return 0;
        s = seq_view(A, i);
        return seq_units<SEL>(A, s);
    }
    __device__ __forceinline__ uint32_t runs_of(uint32_t u) const
    {
        return u ? (u - 1) / per + 1 : 0;
    }
    /* sequences i0 .. i0 + 63, which follow on `before` units, to LDS */
    __device__ __forceinline__ void place(const SeqView &s, uint32_t u, uint32_t before,
                                          uint32_t lane, uint32_t w, RunsLds &L) const
    {
        const uint32_t r = whole ? runs_of(u) * per : u, to = before + scan_wave(r);
        if (w == 0) {
            L.row[lane] = s.part ? s.row : kNone;
            L.lo[lane] = s.lo;
            L.end[lane] = s.end;
            L.units[lane] = u;
            L.from[lane] = to - r;
            L.to[lane] = to;
        }
        __syncthreads();
    }
    __device__ __forceinline__ void begin(const PagesArgs &A, uint32_t lane, uint32_t w, RunsLds &L)
    {
        SeqView s;
        uint32_t u = 0, total = 0;
        runs = 0;
        for (i0 = 0; i0 < A.n_seqs; i0 += 64) {
            u = units(A, i0 + lane, s);
            total += sum_wave(u);
        }
        per = (total + A.share - 1) / A.share;
        per = per > kLeastUnits ? per : kLeastUnits;
        for (i0 = 0; i0 < A.n_seqs; i0 += 64) {
            if (A.n_seqs > 64)
                u = units(A, i0 + lane, s);
            runs += sum_wave(runs_of(u));
        }
        whole = runs <= A.share;
        runs = whole ? runs : (total + per - 1) / per;
        i0 = 0;
        if (A.n_seqs > 64)
            u = units(A, lane, s);
        place(s, u, 0, lane, w, L);
    }
    /* the next 64 sequences; false: there are none */
    __device__ __forceinline__ bool next(const PagesArgs &A, uint32_t lane, uint32_t w, RunsLds &L)
    {
        if (i0 + 64 >= A.n_seqs)
            return false;
        const uint32_t before = L.to[63];
        __syncthreads();
        i0 += 64;
        SeqView s;
        const uint32_t u = units(A, i0 + lane, s);
        place(s, u, before, lane, w, L);
        return true;
    }
};

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

/* waves a SIMD that an instance keeps its registers for, and with that the
   workgroups a compute unit holds. f16 rows up to 128 stream faster with 3 than
   with the 4 that fit (60 sequences at 4170 positions 165.4 -> 159.8 us; 2: 157.8,
   but 100 sequences of up to 500 positions 29.9 -> 31.1); int8 rows, half as many
   bytes in flight a wave, with 4 (32 to 8k 57.3, with 3 62.1), and at 512 with 2
   (60 000 positions, 16 / 2 heads: 41.5 -> 34.5 against 1) */
constexpr int pages_waves(int kv, int d)
{
    if (kv == kF32)
        return d <= 64 ? 4 : d <= 128 ? 2 : 1;
    if (d <= 128)
        return d <= 64 || kv == kI8 ? 4 : kv == kF16 ? 3 : 2;
    if (d <= 256)
        return kv == kI8 ? 3 : 2;
    return kv == kI8 ? 2 : 1;
}

/* units that a wave holds: two where rows of 64 bytes would leave too few bytes in
   flight (32 sequences to 20k, 12 / 4 / 64 int8: 48.4 -> 40.3 us) or, at two waves
   a SIMD, int16's many steps between loads (16 to 8k, 32 / 8 / 128: 55.7 -> 53.6).
   Elsewhere the registers cost more than they bring: f32 at 256 59.6 -> 73.4, f16
   and int16 at 64 a hundredth longer, no gain for f16 or int8 at 128 */
constexpr int pages_buffers(int kv, int d)
{
    return (d == 64 && kv == kI8) || (d == 128 && kv == kI16) ? 2 : 1;
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
    /* the query's operands stay in registers; from head size 256 on they are read
       from LDS at each use: they would cost a wave a SIMD (256) or spill (512) */
    static constexpr bool QREG = D < 256;
    static constexpr int QROW = F32 ? D + 4 : D / 2 + 4; /* words of an LDS row */
    static constexpr int WAVES = pages_waves(T, D);  /* a SIMD, by registers */
    static constexpr int NB = pages_buffers(T, D);
};

template <bool KEEP, class V> __device__ __forceinline__ V load_once(const V *p)
{
    return KEEP ? *p : __builtin_nontemporal_load(p);
}

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

/* MULTI: a KV head's query rows take several workgroups, which read the same
   keys and values: they are dealt to one XCD, side by side, and keep them in its
   L2. Else every row is read once, past the caches (60 sequences at 4170
   positions 187 -> 168 us; 32 query heads on one KV head, with the caches,
   53.7 -> 45.4). */
template <int T, int D, bool SEL, bool MULTI>
__global__ __launch_bounds__(kPW * 64)
__attribute__((amdgpu_waves_per_eu(PS<T, D>::WAVES))) void pages_kernel(const PagesArgs A)
{
    using S = PS<T, D>;
    constexpr int EB = S::EB, KL = S::KL, VN = S::VN, VU = S::VU, VW = S::VW, NT = S::NT;
    constexpr int DP = S::DP, ROWS = S::ROWS, NB = S::NB;
    constexpr bool F32 = S::F32, SCALED = S::SCALED;
    /* where a K row's loads lie is found anew for each unit, not kept in up to 16
       registers (f32, 16 x 4000 positions of 16 / 4 / 256: 58.7 -> 57.8 us; int8 at
       512 has room for a second wave a SIMD with it; not for int16 at 512, 76.0 ->
       77.9, whose registers hold) */
    constexpr bool LEAN = (F32 && D == 256) || (T == kI8 && D == 512);
    typedef typename Words<VW>::T VT;
    /* the query's operands, and the waves' sums: from head size 256 on in the same
       place */
    constexpr bool QREG = S::QREG;
    struct Apart {
        float o[kPW][ROWS][D], q[16][S::QROW];
    };
    union Shared {
        float o[kPW][ROWS][D], q[16][S::QROW];
    };
    __shared__ __attribute__((aligned(16))) typename std::conditional<QREG, Apart, Shared>::type sX;
    auto &sO = sX.o;
    auto &sQ = sX.q;
    __shared__ float sM[kPW][ROWS], sL[kPW][ROWS];
    __shared__ float sE[kPW];
    __shared__ float sQs[ROWS];
    __shared__ RunsLds sR;

    const uint32_t thread = threadIdx.x, w = __builtin_amdgcn_readfirstlane(thread >> 6);
    /* with more than 64 sequences, one workgroup more, the first, writes the plan;
       else the first does it besides */
    const bool planner = A.n_seqs > 64;
    uint32_t run = blockIdx.z - (planner ? 1 : 0), kvh = blockIdx.y, rt = blockIdx.x;
    Runs<SEL> R;
    R.begin(A, thread & 63, w, sR);
    if (blockIdx.x + blockIdx.y + blockIdx.z == 0) {
        /* for the merge, each sequence's partials: the one of run x and sequence
           i has number x + i */
        const uint32_t lane = thread & 63;
        do {
            const uint32_t i = R.i0 + lane, u = sR.units[lane];
            const uint32_t r0 = sR.from[lane] / R.per;
            const uint32_t r1 = u ? (sR.from[lane] + u - 1) / R.per + 1 : r0;
            if (w == kPW - 1 && i < A.n_seqs)
                A.plan[i] = make_uint2(r0 + i, sR.row[lane] == kNone ? kNone : r1 - r0);
        } while (R.next(A, lane, w, sR));
    }
    if (planner && blockIdx.z == 0)
        return;
    const uint32_t tiles = A.n_kv * A.rtiles;
    if constexpr (MULTI) {
        const uint32_t all = R.runs * tiles, id = (run * A.n_kv + kvh) * A.rtiles + rt;
        if (id >= all)
            return;
        const uint32_t to = xcd_remap(id, all);
        rt = to % A.rtiles;
        kvh = to / A.rtiles % A.n_kv;
        run = to / tiles;
    }
    const uint32_t tile = kvh * A.rtiles + rt;
    uint32_t x0 = run * R.per;
    const uint32_t x1 = x0 + R.per;
    /* sequence after sequence of the run */
    for (;;) {
        /* (the thread's number unknown to the compiler: what follows from it is made
           anew for each sequence, not kept in registers across them) */
        uint32_t tid = thread;
        asm volatile("" : "+v"(tid));
        const uint32_t lane = tid & 63, g = lane >> 4, n = lane & 15;
        uint64_t hit;
        while ((hit = __ballot(sR.units[lane] && sR.to[lane] > x0)) == 0)
            if (!R.next(A, lane, w, sR))
                return;
        const uint32_t hl = (uint32_t)__builtin_ctzll(hit);
        const uint32_t si = R.i0 + hl;
        const uint32_t su = __builtin_amdgcn_readfirstlane(sR.units[hl]);
        const uint32_t s0 = __builtin_amdgcn_readfirstlane(sR.from[hl]);
        const uint32_t s1 = __builtin_amdgcn_readfirstlane(sR.to[hl]);
        if (s0 >= x1)
            return;
        SeqView sv;
        sv.row = __builtin_amdgcn_readfirstlane(sR.row[hl]);
        sv.lo = __builtin_amdgcn_readfirstlane(sR.lo[hl]);
        sv.end = __builtin_amdgcn_readfirstlane(sR.end[hl]);
        /* its units [ua, ub) are this run's; `only`: all of them */
        const uint32_t ua = x0 > s0 ? x0 - s0 : 0;
        const uint32_t ub = x1 - s0 < su ? x1 - s0 : su;
        const bool only = ua == 0 && ub == su;
        const uint32_t hd = A.hd, G = A.group, rowb = hd * EB;
        const uint32_t r0 = rt * ROWS;
        const uint32_t rows = G - r0 < ROWS ? G - r0 : ROWS;
        const uint32_t page = 1u << A.page_log, upp = page / kUnit, upp_log = A.page_log - 4;

        /* the wave's quarter of them */
        const uint32_t wa = ua + (ub - ua) * w / kPW, wb = ua + (ub - ua) * (w + 1) / kPW;
        /* units counted from the first page of the list */
        const uint32_t u0 = SEL ? 0 : sv.lo / kUnit;
        const uint32_t first = wa + u0, last = wb + u0; /* [first, last) */

        /* ---- pages: lane i holds entry e0 + i of the wave's list - the block's page
           and its number ---- */
        const uint32_t nb = (sv.end + page - 1) >> A.page_log;
        const uint32_t *const trow = A.table + (size_t)si * A.max_pages;
        const uint32_t *const srow = SEL ? A.sel + ((size_t)si * A.n_kv + kvh) * A.n_sel : nullptr;
        uint32_t e0, pid = 0, blk = 0;
        bool bad = false;            /* a page outside the pool */
        auto fetch = [&](uint32_t from) {
            /* (entries behind the run's last one: that one again) */
            const uint32_t lim = ((last > first ? last : su + u0) - 1) >> upp_log;
            const uint32_t e = from + lane < lim ? from + lane : lim;
            blk = SEL ? srow[e] : e;
            /* (a listed block before the window, whose page may be gone, counts
               for as little as one past the end) */
            const bool in = blk < nb && (!SEL || blk >= sv.lo >> A.page_log);
            pid = trow[in ? blk : 0];
            bad |= in && pid >= A.n_pages;
            pid = in && pid < A.n_pages ? pid : 0;
            blk = in ? blk : kNone;
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

        u4 kr[NB][KL];
        VT vr[NB][4][VU];
        f4 ks[NB], vs[NB];
#pragma unroll
        for (int i = 0; i < NB; i++)
            ks[i] = vs[i] = f4{1, 1, 1, 1};
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
        auto load_k = [&](const Unit &x, auto at) {
            constexpr int B = decltype(at)::value;
            const char *const p = (const char *)A.k + x.row * rowb;
            uint32_t kb = 16 * g;
            if constexpr (LEAN)
                asm volatile("" : "+v"(kb));
#pragma unroll
            for (int i = 0; i < KL; i++) {
                uint32_t to = kat[i];
                if constexpr (LEAN) {
                    bool back;
                    to = 64 * i + kb;
                    to = (EB == 1 ? unit_at(to, rowb, back) : to < rowb ? to : 0) + n * rowb;
                }
                kr[B][i] = load_once<MULTI>((const u4 *)(p + to));
            }
            if constexpr (SCALED)
                ks[B] = *(const f4 *)(A.ks + x.row + 4 * g);
        };
        /* value rows that are not in sight are read as the first or last one that is
           (they weigh 0, but what is there may be no number) */
        auto load_v = [&](const Unit &x, auto at) {
            constexpr int B = decltype(at)::value;
            const char *const p = (const char *)A.v + x.row * rowb;
            uint32_t r[4] = {4 * g * rowb, (4 * g + 1) * rowb, (4 * g + 2) * rowb,
                             (4 * g + 3) * rowb};
            if (x.pos < sv.lo || x.pos + kUnit > sv.end) {
                const uint32_t past = sv.end - 1 - x.pos, short_ = sv.lo - x.pos;
                const uint32_t hi = x.pos < sv.end ? (past < 15 ? past : 15) : 0;
                const uint32_t lo = x.pos < sv.lo ? (short_ < 15 ? short_ : 15) : 0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t y = 4 * g + j > lo ? 4 * g + j : lo;
                    r[j] = (y < hi ? y : hi) * rowb;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int u = 0; u < VU; u++)
                    vr[B][j][u] = load_once<MULTI>((const VT *)(p + (r[j] + vat[u])));
            if constexpr (SCALED)
                vs[B] = *(const f4 *)(A.vs + x.row + 4 * g);
        };

        /* ---- the query: MFMA column n's (row n / 2, plane n & 1; f32: row n) as the
           B operand of each K load. Planes: scaled by 2^ex so that the row's
           largest lies in [2^13, 2^14). The workgroup makes them once, 256 / ROWS
           lanes a row, words of four, through LDS; asked for first, made when the
           first unit's keys have been asked for: one round trip for the query and the
           table, one for the unit ---- */
        constexpr int TPR = kPW * 64 / ROWS, NQ = (D + 4 * TPR - 1) / (4 * TPR);
        const uint32_t qrow = tid / TPR;
        const char *const qsrc =
            (const char *)(A.q + (size_t)sv.row * A.q_stride + (size_t)(kvh * G + r0) * hd);
        const uint32_t qat = (qrow < rows ? qrow : 0) * hd;
        f4 qx[NQ];
        uint32_t qc[NQ];
#pragma unroll
        for (int j = 0; j < NQ; j++) {
            qc[j] = 4 * (tid % TPR + TPR * j);
            qx[j] = *(const f4 *)(qsrc + 4 * (qat + (qc[j] < hd ? qc[j] : 0)));
        }
        __builtin_amdgcn_sched_barrier(0);
        /* (a wave without units asks for a whole one all the same: no branch
           holds up what follows) */
        const uint32_t some = first < su + u0 ? first : su + u0 - 1;
        e0 = some >> upp_log;
        fetch(e0);
        Unit x = unit_of(some);
        typedef std::integral_constant<int, 0> First;
        typedef std::integral_constant<int, NB - 1> Second;
        load_k(x, First());

        float qmax = 0.0f;
#pragma unroll
        for (int j = 0; j < NQ; j++) {
            /* (used as loaded: the compiler else loads only where it is kept, in
               a branch, and waits there for everything before it) */
            asm volatile("" : "+v"(qx[j]));
            if (qrow >= rows || qc[j] >= hd)
                qx[j] = f4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 4; e++)
                qmax = fmaxf(qmax, fabsf(qx[j][e]));
        }
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < NQ; j++)
                *(f4 *)&sQ[qrow][qc[j]] = qx[j];
        } else {
            qmax = max_x16(max_row16(qmax)); /* the row's 32 lanes */
            const int ex = plane_exponent(qmax);
            const float up = ldexpf(1.0f, ex), neg1 = minus_one();
#pragma unroll
            for (int j = 0; j < NQ; j++) {
                h2 hi[2], lo[2];
#pragma unroll
                for (int e = 0; e < 2; e++)
                    split_hl2(qx[j][2 * e] * up, qx[j][2 * e + 1] * up, neg1, hi[e], lo[e]);
                if (D >= 128 || qc[j] < D) {
                    *(uint2 *)&sQ[2 * qrow][qc[j] / 2] = make_uint2(
                        __builtin_bit_cast(uint32_t, hi[0]), __builtin_bit_cast(uint32_t, hi[1]));
                    *(uint2 *)&sQ[2 * qrow + 1][qc[j] / 2] = make_uint2(
                        __builtin_bit_cast(uint32_t, lo[0]), __builtin_bit_cast(uint32_t, lo[1]));
                }
            }
            if (tid % TPR == 0)
                sQs[qrow] = ldexpf(1.0f, -ex);
        }
        /* (its values once the planes are made, which wait for the query alone; against
           with the keys: 90k positions of 16 / 2 / 512 int16 76.1 -> 73.7 us, 16 to 16k
           of 16 / 2 / 256 int8 36.2 -> 35.0; f32's, of which the planes are no more than
           a copy, before the others are waited for: 16 to 4k of 256 57.2, after 59.7) */
        if constexpr (F32)
            load_v(x, First());
        __syncthreads();
        if constexpr (!F32)
            load_v(x, First());
        const float qs2 = (F32 ? 1.0f : sQs[n >> 1]) * A.scale * kLog2e;
        constexpr int QO = EB == 1 ? 2 : 1; /* operands a K load */
        auto q_place = [&](int i, int j, uint32_t place) {
            return *(const u4 *)((const char *)&sQ[0][0] + place + 64 * QO * i + 16 * j);
        };
        const uint32_t qplace = n * S::QROW * 4 + 16 * QO * g;
        u4 qr[QREG ? KL : 1][QREG ? QO : 1];
        if constexpr (QREG) {
#pragma unroll
            for (int i = 0; i < KL; i++)
#pragma unroll
                for (int j = 0; j < QO; j++)
                    qr[i][j] = q_place(i, j, qplace);
        }
        /* operand j of K load i; `place`: the lane's in LDS, unknown to the compiler
           from unit to unit, so that the reads stay in the loop */
        auto q_operand = [&](int i, int j, uint32_t place) {
            if constexpr (QREG)
                return qr[i][j];
            else
                return q_place(i, j, place);
        };

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
        /* unit u from buffers `at`; with two, unit u + 1 is asked for whole before it,
           into the others; with one, its keys once this one's are used, its values
           after this one's */
        auto unit = [&](uint32_t u, auto at, auto other) {
            constexpr int B = decltype(at)::value;
            const Unit now = x;
            const bool more = u + 1 < last;
            if (more)
                x = unit_of(u + 1);
            if (NB == 2 && more) {
                load_k(x, other);
                load_v(x, other);
            }
            /* scores: lane holds positions 4 g + j of MFMA column n */
            f4 s{0, 0, 0, 0};
            uint32_t place = qplace;
            if constexpr (!QREG)
                asm volatile("" : "+v"(place));
#pragma unroll
            for (int i = 0; i < KL; i++) {
                /* (else the query's reads for all of them are made first, in
                   registers that are not there: 90k positions of int16, 80.5 ->
                   77.7 us; int8 holds those of one load with two waves a SIMD) */
                if (D > 256 && (T == kI8 || i % 4 == 0))
                    __builtin_amdgcn_sched_barrier(0);
                const u4 q0 = q_operand(i, 0, place);
                if constexpr (F32) {
                    const f4 kf = __builtin_bit_cast(f4, kr[B][i]), qf = __builtin_bit_cast(f4, q0);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[e], s, 0, 0, 0);
                } else if constexpr (T == kI8) {
                    const u4 y = unit_fix(kr[B][i], kback[i]);
                    s = mfma(i8_widen8(y.x, y.y), __builtin_bit_cast(h8, q0), s);
                    const u4 q1 = q_operand(i, 1, place);
                    s = mfma(i8_widen8(y.z, y.w), __builtin_bit_cast(h8, q1), s);
                } else if constexpr (T == kI16) {
                    h8 hi, lo;
                    i16_planes8(kr[B][i].x, kr[B][i].y, kr[B][i].z, kr[B][i].w, hi, lo);
                    s = mfma(hi, __builtin_bit_cast(h8, q0), s);
                    s = mfma(lo, __builtin_bit_cast(h8, q0), s);
                } else {
                    s = mfma(__builtin_bit_cast(h8, kr[B][i]), __builtin_bit_cast(h8, q0), s);
                }
            }
            const f4 kz = ks[B];
            if (NB == 1 && more)
                load_k(x, other);
            if (now.pos < sv.end && now.pos + kUnit > sv.lo) {
                f4 vz = vs[B];
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
                                    pf[j], __uint_as_float(word<VW>(vr[B][j][c], e)), o[t],
                                    0, 0, 0);
                        } else {
                            const VT v4[4] = {vr[B][0][c], vr[B][1][c], vr[B][2][c], vr[B][3][c]};
                            h4 vb[DP];
                            value_operand<T, VW>(v4, e, vb);
#pragma unroll
                            for (int d = 0; d < DP; d++)
                                o[t] = __builtin_amdgcn_mfma_f32_16x16x16f16(pa, vb[d], o[t],
                                                                             0, 0, 0);
                        }
                    }
            }
            if (NB == 1 && more)
                load_v(x, other);
        };
        for (uint32_t u = first; u < last; u += NB) {
            unit(u, First(), Second());
            if (NB == 2 && u + 1 < last)
                unit(u + 1, Second(), First());
        }

        /* ---- the waves joined ---- */
        if constexpr (!QREG)
            __syncthreads();
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
                    *(f4 *)&sO[w][r][16 * VN * c + VN * n + e] =
                        f4{y[e], y[e + 1], y[e + 2], y[e + 3]};
            }
        __syncthreads();
        for (uint32_t t = tid; t < rows * (D / 4); t += kPW * 64) {
            const uint32_t r = t / (D / 4), c = 4 * (t % (D / 4));
            if (c >= hd)
                continue;
            const float mx = fmaxf(fmaxf(sM[0][r], sM[1][r]), fmaxf(sM[2][r], sM[3][r]));
            f4 y{0, 0, 0, 0};
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < kPW; i++) {
                const float mi = sM[i][r];
                const float f = mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - mx);
                sum += f * sL[i][r];
                const f4 x = *(const f4 *)&sO[i][r][c];
                const float fo = f * sE[i];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    y[e] += fo * x[e];
            }
            if (!only) {
                const size_t pr = ((size_t)(run + si) * tiles + tile) * ROWS + r;
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
        x0 = s1;
        if (x0 >= x1)
            return;
        __syncthreads(); /* (the next sequence's rows take the same LDS) */
    }
}

/* ---- the merge --------------------------------------------------------------- */

constexpr int kMBatch = 4;

/*
 * A row's partials joined, COLS columns a workgroup of WAVES waves: COLS / 4 lanes
 * take a partial (a float4 each), so 256 / COLS x WAVES go at once, group i taking
 * partials i, i + groups, ... with a running maximum; the groups of a wave and
 * then the waves are joined in a fixed tree. Rows of one workgroup of
 * pages_kernel's are written there; rows that see nothing are written here: 0, or
 * NaN where the length passes the table.
 *
 * Bound by its launch and two dependent reads: 3.5 to 4.7 us. 32 columns where there are few rows
 * (many partials each, and the device to fill), 128 where there are many
 * (pages_merge_cols), and one wave where a row has few partials.
 */
template <int ROWS, int COLS, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void pages_merge_kernel(const PagesArgs A)
{
    constexpr uint32_t LANES = COLS / 4, GROUPS = WAVES * 64 / LANES;
    __shared__ float sM[WAVES], sL[WAVES];
    __shared__ f4 sA[WAVES][LANES];
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t hd = A.hd, h = blockIdx.y, si = blockIdx.z;
    const uint32_t col = blockIdx.x * COLS + 4 * (lane % LANES);
    const uint2 plan = A.plan[si];
    const uint32_t row = A.row ? A.row[si] : si;
    const uint32_t first = plan.x, count = plan.y;
    if (count == kNone || count == 1)
        return;
    const size_t hr = (size_t)row * A.n_head + h;
    if (count == 0) {
        const float z = A.len[si] > A.max_pages << A.page_log ? NAN : 0.0f;
        if (tid < LANES && col < hd)
            *(f4 *)(A.out + hr * hd + col) = f4{z, z, z, z};
        return;
    }
    const uint32_t kvh = h / A.group, r = h % A.group;
    const uint32_t tiles = A.n_kv * A.rtiles, tile = kvh * A.rtiles + r / ROWS;
    const uint32_t at = col < hd ? col : 0;
    /* the gate, asked for with the partials */
    f4 sg{1, 1, 1, 1};
    if (A.gate_mode == kGateElem)
        sg = *(const f4 *)(A.gate + hr * hd + at);
    else if (A.gate_mode == kGateHead)
        sg[0] = sg[1] = sg[2] = sg[3] = A.gate[hr];
    float m = -INFINITY, l = 0.0f;
    f4 a{0, 0, 0, 0};
    for (uint32_t i0 = tid / LANES; i0 < count; i0 += GROUPS * kMBatch) {
        float2 ml[kMBatch];
        f4 x[kMBatch];
#pragma unroll
        for (int b = 0; b < kMBatch; b++) {
            uint32_t i = i0 + GROUPS * b;
            i = i < count ? i : count - 1;
            const size_t pr = ((size_t)(first + i) * tiles + tile) * ROWS + r % ROWS;
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
            const bool in = i0 + GROUPS * b < count && ml[b].x != -INFINITY;
            const float e = in ? __builtin_amdgcn_exp2f(ml[b].x - mn) : 0.0f;
            l += in ? e * ml[b].y : 0.0f;
#pragma unroll
            for (int c = 0; c < 4; c++)
                a[c] = __builtin_fmaf(e, x[b][c], a[c]);
        }
    }
    /* the wave's groups, then the waves */
    float mw = m;
#pragma unroll
    for (int o = LANES; o < 64; o <<= 1)
        mw = fmaxf(mw, __shfl_xor(mw, o, 64));
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mw);
    l *= f;
    a *= f;
#pragma unroll
    for (int o = LANES; o < 64; o <<= 1) {
        l += __shfl_xor(l, o, 64);
#pragma unroll
        for (int c = 0; c < 4; c++)
            a[c] += __shfl_xor(a[c], o, 64);
    }
    float sum = l;
    f4 y = a;
    if constexpr (WAVES > 1) {
        if (lane == 0) {
            sM[w] = mw;
            sL[w] = l;
        }
        if (lane < LANES)
            sA[w][lane] = a;
        __syncthreads();
        if (tid >= LANES)
            return;
        float mx = sM[0];
#pragma unroll
        for (int i = 1; i < WAVES; i++)
            mx = fmaxf(mx, sM[i]);
        sum = 0.0f;
        y = f4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < WAVES; i++) {
            const float e = sM[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sM[i] - mx);
            sum += e * sL[i];
            y += e * sA[i][lane];
        }
    }
    if (tid >= LANES || col >= hd)
        return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
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
    const dim3 grid(a.rtiles, a.n_kv, a.runs + (a.n_seqs > 64)), block(kPW * 64);
    if (a.sel && a.rtiles > 1)
        hipLaunchKernelGGL((pages_kernel<T, D, true, true>), grid, block, 0, s, a);
    else if (a.sel)
        hipLaunchKernelGGL((pages_kernel<T, D, true, false>), grid, block, 0, s, a);
    else if (a.rtiles > 1)
        hipLaunchKernelGGL((pages_kernel<T, D, false, true>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((pages_kernel<T, D, false, false>), grid, block, 0, s, a);
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

uint32_t pages_share(int kv, uint32_t hd, uint32_t cus, uint32_t tiles)
{
    const uint32_t fill = pages_waves(kv, (int)hd) * cus;
    return fill / tiles > 1 ? fill / tiles : 1;
}

uint64_t pages_runs(uint32_t share, uint32_t n_seqs, uint64_t most_units)
{
    /* no more than the lengths that the table's rows hold can fill */
    return std::min<uint64_t>(share, n_seqs * ((most_units + kLeastUnits - 1) / kLeastUnits));
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

uint32_t pages_merge_cols(uint32_t n_seqs, uint32_t n_head, uint32_t hd)
{
    return hd > 32 && (uint64_t)n_seqs * n_head * ((hd + 127) / 128) >= kMergeFill ? 128 : 32;
}

template <int ROWS, int COLS> static void launch_merge_cols(const PagesArgs &a, hipStream_t s)
{
    const dim3 grid((a.hd + COLS - 1) / COLS, a.n_head, a.n_seqs);
    /* a row's partials are about a sequence's share of the runs: a wave's batch
       holds 4 x 256 / COLS of them */
    if (a.share <= a.n_seqs * kMBatch * (256 / COLS))
        hipLaunchKernelGGL((pages_merge_kernel<ROWS, COLS, 1>), grid, dim3(64), 0, s, a);
    else
        hipLaunchKernelGGL((pages_merge_kernel<ROWS, COLS, 4>), grid, dim3(256), 0, s, a);
}

hipError_t launch_pages_merge(int kv, const PagesArgs &a, hipStream_t s)
{
    const bool wide = pages_merge_cols(a.n_seqs, a.n_head, a.hd) == 128;
    if (kv == kF32 && wide)
        launch_merge_cols<16, 128>(a, s);
    else if (kv == kF32)
        launch_merge_cols<16, 32>(a, s);
    else if (wide)
        launch_merge_cols<8, 128>(a, s);
    else
        launch_merge_cols<8, 32>(a, s);
    return hipGetLastError();
}

}  // namespace janas
