/*
 * attn_pages_api.cpp - Part 4 of include/janas_attn.h: the paged cache's entry
 * points over the kernels of attn_pages.hip, attn_pages_plan.hip,
 * attn_pages_select.hip and the paged rows of attn_cache.hip.
 */
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include <hip/hip_runtime.h>

#include "../../include/janas_attn.h"
#include "attn_kernels.h"
#include "attn_pages.h"

using namespace janas;

namespace {

int hip_rc(hipError_t e, const char *what)
{
    if (e == hipSuccess)
        return JANAS_ATTN_OK;
    fprintf(stderr, "janas_attn: %s: %s\n", what, hipGetErrorString(e));
    return JANAS_ATTN_EDEVICE;
}

/* The pool's device for the launches of a call, and the caller's again after */
struct OnDevice {
    int was = -1, rc = JANAS_ATTN_OK;
    explicit OnDevice(int dev)
    {
        int now = -1;
        rc = hip_rc(hipGetDevice(&now), "get device");
        if (rc || now == dev)
            return;
        rc = hip_rc(hipSetDevice(dev), "set device");
        if (!rc)
            was = now;
    }
    ~OnDevice()
    {
        if (was >= 0)
            (void)hipSetDevice(was);
    }
};

bool aligned(const void *p, size_t bytes) { return (uintptr_t)p % bytes == 0; }

uint32_t log2_of(uint32_t x) { return (uint32_t)__builtin_ctz(x); }

constexpr uint64_t kMostSlots = 1ull << 31;
/* a launch's threads count in 32 bits */
constexpr uint64_t kMostThreads = 0xFFFFFFFFull;

int check_tables(const janas_attn_pages *p)
{
    if (!p || !p->table || !p->len || p->dev < 0 || p->page < 16 || p->page > 256 ||
        (p->page & (p->page - 1)) || p->n_pages == 0 || p->n_seqs == 0 || p->n_seqs > 65535 ||
        p->max_pages == 0)
        return JANAS_ATTN_EINVAL;
    if ((uint64_t)p->n_pages * p->page >= kMostSlots ||
        (uint64_t)p->max_pages * p->page >= kMostSlots)
        return JANAS_ATTN_ERANGE;
    return JANAS_ATTN_OK;
}

int check_pool(const janas_attn_pages *p)
{
    int rc = check_tables(p);
    if (rc)
        return rc;
    if (!p->k || !p->v || p->n_kv == 0 || p->n_kv > 65535 || p->head_dim == 0 ||
        p->head_dim > 512 || p->head_dim % 8 || p->kv_type < kI8 || p->kv_type > kF32)
        return JANAS_ATTN_EINVAL;
    if ((p->kv_type == kI8 || p->kv_type == kI16) && (!p->ks || !p->vs))
        return JANAS_ATTN_EINVAL;
    if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->ks, 16) || !aligned(p->vs, 16) ||
        !aligned(p->bounds, 16))
        return JANAS_ATTN_EINVAL;
    return JANAS_ATTN_OK;
}

/* an instance over a pool */
int check_instance(const janas_attn *a, const janas_attn_pages *p)
{
    if (!a)
        return JANAS_ATTN_EINVAL;
    int rc = check_pool(p);
    if (rc)
        return rc;
    const PagesGeom g = pages_geom(a);
    if (g.n_kv != p->n_kv || g.hd != p->head_dim || g.dev != p->dev)
        return JANAS_ATTN_EINVAL;
    if (g.ring || !pages_supported(p->kv_type, p->head_dim))
        return JANAS_ATTN_ENOTSUP;
    return JANAS_ATTN_OK;
}

/* a call's single tokens: their queries and which sequences take part */
int check_rows(const PagesGeom &g, const janas_attn_pages_call *c)
{
    const uint64_t width = (uint64_t)g.n_head * g.hd;
    if (!c || !c->q || !aligned(c->q, 16) || c->q_stride % 4 ||
        (c->q_stride && c->q_stride < width) || !c->row != !c->granted ||
        !aligned(c->work, 256))
        return JANAS_ATTN_EINVAL;
    return JANAS_ATTN_OK;
}

/* no rows, so that no sequence takes part */
bool no_rows(const janas_attn_pages_call *c)
{
    return c && c->row && c->granted && c->n_rows == 0;
}

/* the runs of a call and the bytes of their partials */
struct Parts {
    uint32_t rtiles, share;
    uint64_t runs, plan_bytes, ml_bytes, bytes;
};
Parts parts_of(const PagesGeom &g, const janas_attn_pages *p)
{
    Parts t;
    const uint32_t rows = pages_rows_wg(p->kv_type);
    t.rtiles = (g.group + rows - 1) / rows;
    const uint32_t tiles = g.n_kv * t.rtiles;
    t.share = pages_share(p->kv_type, g.hd, g.cus, tiles);
    t.runs = pages_runs(t.share, p->n_seqs, (uint64_t)p->max_pages * p->page / 16);
    const uint64_t parts = (t.runs + p->n_seqs) * tiles * rows;
    t.plan_bytes = ((uint64_t)p->n_seqs * sizeof(uint2) + 255) / 256 * 256;
    t.ml_bytes = (parts * 2 * sizeof(float) + 255) / 256 * 256;
    t.bytes = t.plan_bytes + t.ml_bytes + parts * g.hd * sizeof(float);
    return t;
}

uint64_t score_bytes(const janas_attn_pages *p)
{
    return (uint64_t)p->n_seqs * p->n_kv * p->max_pages * sizeof(float);
}

/* whether the pool's and the instance's sizes alone let janas_attn_pages_run ... */
int run_fits(const PagesGeom &g, const janas_attn_pages *p, const Parts &t)
{
    if ((uint64_t)g.n_head * g.hd > 0xFFFFFFFFu || g.n_head > 65535)
        return JANAS_ATTN_ERANGE;
    /* a call's units of 16 positions in 32 bits, with what rounds them up and times
       the four waves that share them */
    if ((uint64_t)p->n_seqs * p->max_pages * (p->page / 16) >= 1ull << 30)
        return JANAS_ATTN_ERANGE;
    const uint64_t cols = pages_merge_cols(p->n_seqs, g.n_head, g.hd);
    const uint64_t merge_wg = (uint64_t)p->n_seqs * g.n_head * ((g.hd + cols - 1) / cols);
    return std::max((t.runs + 1) * g.n_kv * t.rtiles, merge_wg) > kMostThreads / 256
               ? JANAS_ATTN_ERANGE
               : JANAS_ATTN_OK;
}

/* ... and janas_attn_pages_select take them */
int select_fits(const PagesGeom &g, const janas_attn_pages *p)
{
    return (uint64_t)g.n_head * g.hd > 0xFFFFFFFFu || p->max_pages > 1u << 20 ||
                   (uint64_t)p->n_seqs * p->n_kv > kMostThreads / 1024
               ? JANAS_ATTN_ERANGE
               : JANAS_ATTN_OK;
}

}  // namespace

extern "C" int janas_attn_pages_plan(const struct janas_attn_pages *p,
                                     const struct janas_attn_plan *s,
                                     void *stream)
{
    int rc = check_tables(p);
    if (rc)
        return rc;
    if (!s || !p->free_pages || !p->n_free || !s->n_new || !s->len || !s->n_free || !s->granted ||
        !s->start || !s->taken || (s->max_tokens && (!s->slot || !s->pos || !s->seq)))
        return JANAS_ATTN_EINVAL;
    if (s->max_tokens >= kMostSlots)
        return JANAS_ATTN_ERANGE;
    PlanArgs a;
    memset(&a, 0, sizeof a);
    a.table = p->table;
    a.len = p->len;
    a.n_free = p->n_free;
    a.n_new = s->n_new;
    a.free_pages = p->free_pages;
    a.len_out = s->len;
    a.n_free_out = s->n_free;
    a.granted = s->granted;
    a.start = s->start;
    a.taken = s->taken;
    a.slot = s->slot;
    a.pos = s->pos;
    a.seq = s->seq;
    a.n_seqs = p->n_seqs;
    a.max_pages = p->max_pages;
    a.n_pages = p->n_pages;
    a.page_log = log2_of(p->page);
    a.max_tokens = s->max_tokens;
    OnDevice on(p->dev);
    return on.rc ? on.rc : hip_rc(launch_plan(a, (hipStream_t)stream), "plan launch");
}

extern "C" int janas_attn_pages_write(const struct janas_attn_pages *p,
                                      const struct janas_attn_rows *r,
                                      void *stream)
{
    int rc = check_pool(p);
    if (rc)
        return rc;
    const uint32_t hd = p->head_dim;
    if (r && r->n == 0)
        return JANAS_ATTN_OK; /* (an empty tensor has no address) */
    if (!r || !r->k || !r->v || !r->slot || r->n_rot % 2 || r->n_rot > hd ||
        (r->n_rot && (!r->cs || !r->sn || !r->pos || r->n_tab == 0)) ||
        (r->q && (!r->q_out || r->n_head == 0)))
        return JANAS_ATTN_EINVAL;
    const uint64_t kw = (uint64_t)p->n_kv * hd, qw = r->q ? (uint64_t)r->n_head * hd : 0;
    if (kw > 0xFFFFFFFFu || qw > 0xFFFFFFFFu)
        return JANAS_ATTN_ERANGE;
    if ((r->k_stride && r->k_stride < kw) || (r->v_stride && r->v_stride < kw) ||
        (r->q && r->q_stride && r->q_stride < qw) ||
        (r->q && r->q == r->q_out && r->q_stride && r->q_stride != qw))
        return JANAS_ATTN_EINVAL;
    PagesRowArgs a;
    memset(&a, 0, sizeof a);
    a.k = r->k;
    a.v = r->v;
    a.q = r->q;
    a.q_out = r->q_out;
    a.k_norm = r->k_norm;
    a.q_norm = r->q_norm;
    a.cs = r->cs;
    a.sn = r->sn;
    a.kc = p->k;
    a.vc = p->v;
    a.kz = p->ks;
    a.vz = p->vs;
    a.slot = r->slot;
    a.pos = r->pos;
    a.inv_hd = 1.0 / hd;
    a.eps = r->eps;
    a.n = r->n;
    a.n_kv = p->n_kv;
    a.n_head = r->q ? r->n_head : 0;
    a.hd = hd;
    a.n_rot = r->n_rot;
    a.n_tab = r->n_tab;
    a.k_stride = r->k_stride ? r->k_stride : (uint32_t)kw;
    a.v_stride = r->v_stride ? r->v_stride : (uint32_t)kw;
    a.q_stride = r->q_stride ? r->q_stride : (uint32_t)qw;
    a.page_log = log2_of(p->page);
    a.n_slots = p->n_pages << a.page_log;
    a.kv = p->kv_type;
    a.v_norm = r->v_norm != 0;
    /* a row takes a wave at most */
    if ((uint64_t)a.n * ((uint64_t)a.n_kv + a.n_head) > kMostThreads / 64 - 4)
        return JANAS_ATTN_ERANGE;
    OnDevice on(p->dev);
    return on.rc ? on.rc : hip_rc(launch_pages_rows(a, (hipStream_t)stream), "page rows launch");
}

extern "C" int janas_attn_pages_bounds(const struct janas_attn_pages *p,
                                       const uint32_t *n_new, uint32_t max_new,
                                       void *stream)
{
    int rc = check_pool(p);
    if (rc)
        return rc;
    if (!p->bounds)
        return JANAS_ATTN_EINVAL;
    BoundsArgs a;
    memset(&a, 0, sizeof a);
    a.k = p->k;
    a.ks = p->kv_type == kI8 || p->kv_type == kI16 ? p->ks : nullptr;
    a.bounds = (_Float16 *)p->bounds;
    a.table = p->table;
    a.len = p->len;
    a.n_new = n_new;
    a.n_seqs = p->n_seqs;
    a.n_kv = p->n_kv;
    a.hd = p->head_dim;
    a.max_pages = p->max_pages;
    a.n_pages = p->n_pages;
    a.page_log = log2_of(p->page);
    a.kv = p->kv_type;
    /* a workgroup of each at least, for every 128 columns */
    if ((uint64_t)p->n_seqs * p->n_kv * bound_slices(a.hd) > kMostThreads / 256)
        return JANAS_ATTN_ERANGE;
    /* the blocks that max_new positions may touch; a workgroup goes on to
       further ones (2^20 x 4 workgroups or one a block's slice: a launch holds
       them) */
    uint64_t blocks = p->max_pages;
    if (n_new && max_new)
        blocks = std::min<uint64_t>(blocks, ((uint64_t)max_new + p->page - 2) / p->page + 1);
    const uint64_t most = std::max<uint64_t>(1, (1u << 20) / ((uint64_t)p->n_seqs * p->n_kv));
    a.max_blocks = (uint32_t)std::min(blocks, most);
    OnDevice on(p->dev);
    return on.rc ? on.rc : hip_rc(launch_bounds(a, (hipStream_t)stream), "key bounds launch");
}

extern "C" size_t janas_attn_pages_work_bytes(const struct janas_attn *a,
                                              const struct janas_attn_pages *p)
{
    if (check_instance(a, p))
        return 0;
    const PagesGeom g = pages_geom(a);
    const Parts t = parts_of(g, p);
    if (run_fits(g, p, t) || (p->bounds && select_fits(g, p)))
        return 0;
    return (size_t)(p->bounds ? std::max(t.bytes, score_bytes(p)) : t.bytes);
}

extern "C" int janas_attn_pages_run(struct janas_attn *a,
                                    const struct janas_attn_pages *p,
                                    int gate_mode,
                                    const struct janas_attn_pages_call *c,
                                    void *stream)
{
    int rc = check_instance(a, p);
    if (rc)
        return rc;
    if (no_rows(c))
        return JANAS_ATTN_OK;
    const PagesGeom g = pages_geom(a);
    rc = check_rows(g, c);
    if (rc)
        return rc;
    if (!c->out || !aligned(c->out, 16) || !c->work || gate_mode < kGateNone ||
        gate_mode > kGateHead || (gate_mode != kGateNone && !c->gate) ||
        (gate_mode == kGateElem && !aligned(c->gate, 16)) || (c->sel && c->n_sel == 0) ||
        (c->out_q8k && (uint64_t)g.n_head * g.hd % JANAS_ATTN_QK))
        return JANAS_ATTN_EINVAL;
    const Parts t = parts_of(g, p);
    rc = run_fits(g, p, t);
    if (rc)
        return rc;
    const uint64_t rows = c->row ? c->n_rows : p->n_seqs;
    const uint64_t blocks = rows * g.n_head * g.hd / JANAS_ATTN_QK;
    if ((c->out_q8k && blocks > kMostThreads / 256) || c->work_bytes < t.bytes)
        return JANAS_ATTN_ERANGE;
    PagesArgs s;
    memset(&s, 0, sizeof s);
    s.k = p->k;
    s.v = p->v;
    s.ks = p->ks;
    s.vs = p->vs;
    s.table = p->table;
    s.len = p->len;
    s.row = c->row;
    s.granted = c->granted;
    s.sel = c->sel;
    s.q = c->q;
    s.gate = c->gate;
    s.out = c->out;
    s.plan = (uint2 *)c->work;
    s.part_ml = (float *)((char *)c->work + t.plan_bytes);
    s.part_acc = (float *)((char *)c->work + t.plan_bytes + t.ml_bytes);
    s.n_seqs = p->n_seqs;
    s.n_rows = c->n_rows;
    s.max_pages = p->max_pages;
    s.n_pages = p->n_pages;
    s.page_log = log2_of(p->page);
    s.n_sel = c->n_sel;
    s.n_head = g.n_head;
    s.n_kv = g.n_kv;
    s.group = g.group;
    s.hd = g.hd;
    s.window = g.window;
    s.q_stride = c->q_stride ? c->q_stride : g.n_head * g.hd;
    s.rtiles = t.rtiles;
    s.share = t.share;
    s.runs = (uint32_t)t.runs;
    s.scale = g.scale;
    s.gate_mode = gate_mode;
    OnDevice on(p->dev);
    if (on.rc)
        return pages_note(a, on.rc);
    rc = hip_rc(launch_pages(p->kv_type, s, (hipStream_t)stream), "pages launch");
    if (!rc)
        rc = hip_rc(launch_pages_merge(p->kv_type, s, (hipStream_t)stream), "pages merge launch");
    if (!rc && c->out_q8k) {
        Q8kArgs q;
        q.x = c->out;
        q.y = (uint8_t *)c->out_q8k;
        q.blocks = (uint32_t)blocks;
        rc = hip_rc(launch_q8k(q, (hipStream_t)stream), "q8k launch");
    }
    return pages_note(a, rc);
}

extern "C" int janas_attn_pages_select(struct janas_attn *a,
                                       const struct janas_attn_pages *p,
                                       const struct janas_attn_pages_call *c,
                                       uint32_t first, uint32_t last,
                                       uint32_t *sel, void *stream)
{
    int rc = check_instance(a, p);
    if (rc)
        return rc;
    if (no_rows(c))
        return JANAS_ATTN_OK;
    const PagesGeom g = pages_geom(a);
    rc = check_rows(g, c);
    if (rc)
        return rc;
    if (!p->bounds || !sel || !c->work || c->n_sel == 0 || (uint64_t)first + last > c->n_sel)
        return JANAS_ATTN_EINVAL;
    rc = select_fits(g, p);
    if (rc)
        return rc;
    if (c->work_bytes < score_bytes(p))
        return JANAS_ATTN_ERANGE;
    SelectArgs s;
    memset(&s, 0, sizeof s);
    s.bounds = (const _Float16 *)p->bounds;
    s.table = p->table;
    s.len = p->len;
    s.row = c->row;
    s.granted = c->granted;
    s.q = c->q;
    s.score = (float *)c->work;
    s.sel = sel;
    s.n_seqs = p->n_seqs;
    s.n_rows = c->n_rows;
    s.n_head = g.n_head;
    s.n_kv = g.n_kv;
    s.group = g.group;
    s.hd = g.hd;
    s.window = g.window;
    s.q_stride = c->q_stride ? c->q_stride : g.n_head * g.hd;
    s.max_pages = p->max_pages;
    s.n_pages = p->n_pages;
    s.page_log = log2_of(p->page);
    s.n_sel = c->n_sel;
    s.first = first;
    s.last = last;
    s.cus = g.cus;
    s.negate = g.scale < 0.0f;
    OnDevice on(p->dev);
    if (on.rc)
        return pages_note(a, on.rc);
    return pages_note(a, hip_rc(launch_select(s, (hipStream_t)stream), "select launch"));
}
