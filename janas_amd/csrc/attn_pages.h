/*
 * attn_pages.h - launch descriptors of the paged cache's kernels
 * (attn_pages.hip, attn_pages_plan.hip, attn_pages_select.hip and the paged
 * rows of attn_cache.hip) and what attn_pages_api.cpp needs of an instance.
 * Internal: not part of the C ABI (include/janas_attn.h, Part 4).
 */
#ifndef JANAS_AMD_ATTN_PAGES_H
#define JANAS_AMD_ATTN_PAGES_H

#include <stdint.h>

#include <hip/hip_runtime.h>

#include "attn_kernels.h"

struct janas_attn;

namespace janas {

constexpr uint32_t kRelease = 0xFFFFFFFFu, kNone = 0xFFFFFFFFu;

/* What the paged calls use of an instance (attn_api.cpp) */
struct PagesGeom {
    uint32_t n_head, n_kv, group, hd, window, cus;
    float scale;
    int ring, dev;
};
PagesGeom pages_geom(const janas_attn *a);
/* a device failure kept in the instance (janas_attn_status); returns rc */
int pages_note(janas_attn *a, int rc);

/* One step of the tables (attn_pages_plan.hip): struct janas_attn_pages and
   janas_attn_plan as the kernels see them */
struct PlanArgs {
    uint32_t *table;
    const uint32_t *len, *n_free, *n_new;
    uint32_t *free_pages;
    uint32_t *len_out, *n_free_out, *granted, *start, *taken;
    uint32_t *slot, *pos, *seq;
    uint32_t n_seqs, max_pages, n_pages, page_log, max_tokens;
    uint32_t whole;        /* plan_kernel writes tables and slots too */
};
hipError_t launch_plan(PlanArgs a, hipStream_t s);

/* A step's rows into their slots (attn_cache.hip) */
struct PagesRowArgs {
    const float *k, *v, *q;
    float *q_out;
    const float *k_norm, *q_norm, *cs, *sn;
    void *kc, *vc;
    float *kz, *vz;
    const uint32_t *slot, *pos;
    double inv_hd;
    float eps;
    uint32_t n, n_kv, n_head, hd, n_rot, n_tab;
    uint32_t k_stride, v_stride, q_stride;
    uint32_t page_log, n_slots;
    int kv, v_norm;
};
hipError_t launch_pages_rows(const PagesRowArgs &a, hipStream_t s);

/* Attention of one token a sequence over its pages (attn_pages.hip) */
struct PagesArgs {
    const void *k, *v;
    const float *ks, *vs;
    const uint32_t *table, *len, *row, *granted, *sel;
    const float *q, *gate;
    float *out;
    float *part_ml;        /* [runs + n_seqs][tiles][rows a workgroup][2] */
    float *part_acc;       /* the same of [hd]; tiles = n_kv x rtiles */
    uint2 *plan;           /* [n_seqs]: a sequence's first partial and their
                              count (kNone: it takes no part) */
    uint32_t n_seqs, n_rows, max_pages, n_pages, page_log, n_sel;
    uint32_t n_head, n_kv, group, hd, window, q_stride;
    uint32_t rtiles;       /* workgroups along a KV head's query rows */
    uint32_t share;        /* runs of a tile that the device holds at once */
    uint32_t runs;         /* pages_runs: workgroups of a tile */
    float scale;
    int gate_mode;
};
/* query rows a workgroup takes */
inline uint32_t pages_rows_wg(int kv) { return kv == kF32 ? 16 : 8; }
int pages_supported(int kv, uint32_t hd);
/* the runs of one of `tiles` = n_kv x rtiles that the device holds at once, and
   the most that a call makes of them (most_units: a table row's) */
uint32_t pages_share(int kv, uint32_t hd, uint32_t cus, uint32_t tiles);
uint64_t pages_runs(uint32_t share, uint32_t n_seqs, uint64_t most_units);
/* columns a merge workgroup takes */
uint32_t pages_merge_cols(uint32_t n_seqs, uint32_t n_head, uint32_t hd);
hipError_t launch_pages(int kv, const PagesArgs &a, hipStream_t s);
hipError_t launch_pages_merge(int kv, const PagesArgs &a, hipStream_t s);

/* Key bounds, scores and the selection (attn_pages_select.hip) */
struct BoundsArgs {
    const void *k;
    const float *ks;
    _Float16 *bounds;
    const uint32_t *table, *len, *n_new;
    uint32_t n_seqs, n_kv, hd, max_pages, n_pages, page_log, max_blocks;
    int kv;
};
/* columns a workgroup takes, and with that the workgroups a block and KV head */
constexpr uint32_t kBoundCols = 128;
__host__ __device__ constexpr uint32_t bound_slices(uint32_t hd)
{
    return (hd + kBoundCols - 1) / kBoundCols;
}
hipError_t launch_bounds(const BoundsArgs &a, hipStream_t s);
struct SelectArgs {
    const _Float16 *bounds;
    const uint32_t *table, *len, *row, *granted;
    const float *q;
    float *score;          /* [n_seqs][n_kv][max_pages] */
    uint32_t *sel;
    uint32_t n_seqs, n_rows, n_head, n_kv, group, hd, window, q_stride;
    uint32_t max_pages, n_pages, page_log, n_sel, first, last, cus;
    int negate;
};
hipError_t launch_select(const SelectArgs &a, hipStream_t s);

/* Sequence i of a call over single tokens, as every kernel of it sees it */
struct SeqView {
    uint32_t row;          /* of q and out */
    uint32_t lo, end;      /* positions in sight */
    bool part, bad;        /* it takes part; its length passes the table */
};
template <class Args>
__device__ __forceinline__ SeqView seq_view(const Args &A, uint32_t i)
{
    SeqView s;
    const uint32_t len = A.len[i], cap = A.max_pages << A.page_log;
    s.row = i;
    s.part = true;
    if (A.row) {
        s.row = A.row[i];
        s.part = A.granted[i] == 1 && s.row < A.n_rows;
    }
    s.bad = len > cap;
    s.end = s.bad ? cap : len;
    s.lo = A.window && len > A.window ? len - A.window : 0;
    s.lo = s.lo < s.end ? s.lo : s.end;
    return s;
}

}  // namespace janas

#endif
