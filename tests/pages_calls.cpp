/*
 * The host side of the paged calls that take an instance, over a made-up
 * instance and device: no GPU and no kernel, device memory is never touched.
 * Loaded as a library (test_pages_limits.py); what the kernels' own sizes
 * depend on comes from the library that it is linked with.
 */
#include "../janas_amd/csrc/attn_pages_api.cpp"

struct janas_attn {
    PagesGeom g;
};
static janas_attn instance;
static int launches;

extern "C" {
struct janas_attn *made_up(uint32_t n_head, uint32_t n_kv, uint32_t hd, int ring)
{
    instance.g = PagesGeom{n_head, n_kv, n_head / n_kv, hd, 0, 256, 0.125f, ring, 0};
    return &instance;
}
int launched(void) { return launches; }

hipError_t hipGetDevice(int *d)
{
    *d = 0;
    return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "refused"; }
}

namespace janas {
PagesGeom pages_geom(const janas_attn *a) { return a->g; }
int pages_note(janas_attn *, int rc) { return rc; }
static hipError_t count()
{
    launches++;
    return hipSuccess;
}
hipError_t launch_plan(PlanArgs, hipStream_t) { return count(); }
hipError_t launch_pages_rows(const PagesRowArgs &, hipStream_t) { return count(); }
hipError_t launch_pages(int, const PagesArgs &, hipStream_t) { return count(); }
hipError_t launch_pages_merge(int, const PagesArgs &, hipStream_t) { return count(); }
hipError_t launch_bounds(const BoundsArgs &, hipStream_t) { return count(); }
hipError_t launch_select(const SelectArgs &, hipStream_t) { return count(); }
hipError_t launch_q8k(const Q8kArgs &, hipStream_t) { return count(); }
}  // namespace janas
