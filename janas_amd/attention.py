"""Python mirror of the engine's attention interface, over libjanas_attn.so.

``Attention`` follows the reference's C API (src/llm/attention.h:58-112)
name for name - create / set_scale / set_window / set_kv16 / set_ring /
set_last / scores_mode / scores_auto / run / destroy - and adds the device
extension of include/janas_attn.h (``run_dev``: f16 / f32 / int8 / int16
caches, several sequences, the fused gate, a stream).

Arrays may be numpy arrays (host memory: janas_attn_run stages them through
the device, as the C entry point does) or anything with ``data_ptr()``
(torch tensors on the GPU: used in place). There is no CPU path: without the
built library this module raises on import of the library.
"""
import ctypes
import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB_PATH = os.path.join(HERE, "libjanas_attn.so")
HEADER = os.path.join(ROOT, "include", "janas_attn.h")

MAX_BLOCK = 64
AUTO, FLOAT, INT16 = 0, 1, 2
KV_I8, KV_I16, KV_F16, KV_F32 = 0, 1, 2, 3
GATE_NONE, GATE_ELEM, GATE_HEAD = 0, 1, 2
ERRORS = {0: "ok", -1: "EINVAL", -2: "ERANGE", -3: "ENOMEM", -4: "EDEVICE",
          -5: "ENOTSUP"}
OK, EINVAL, ERANGE, ENOMEM, EDEVICE, ENOTSUP = 0, -1, -2, -3, -4, -5

_u32 = ctypes.c_uint32
_vp = ctypes.c_void_p


class Seq(ctypes.Structure):
    """struct janas_attn_seq (include/janas_attn.h)."""
    _fields_ = [("k", _vp), ("v", _vp), ("ks", _vp), ("vs", _vp),
                ("q", _vp), ("out", _vp), ("gate", _vp), ("last", _vp),
                ("cap", _u32), ("n", _u32), ("pos0", _u32),
                ("last_max", _u32), ("out_q8k", _vp)]


class Cache(ctypes.Structure):
    """struct janas_attn_cache (include/janas_attn.h Part 3)."""
    _fields_ = [("k", _vp), ("v", _vp), ("ks", _vp), ("vs", _vp),
                ("n_kv", _u32), ("head_dim", _u32), ("cap", _u32),
                ("kv_type", ctypes.c_int), ("ring", ctypes.c_int)]


Q8K_BYTES = 628  # struct janas_attn_q8k
RELEASE = NONE = 0xFFFFFFFF  # -1 in an int32 tensor


class Pages(ctypes.Structure):
    """struct janas_attn_pages (include/janas_attn.h Part 4)."""
    _fields_ = [("k", _vp), ("v", _vp), ("ks", _vp), ("vs", _vp),
                ("bounds", _vp), ("n_kv", _u32), ("head_dim", _u32),
                ("kv_type", ctypes.c_int), ("page", _u32), ("n_pages", _u32),
                ("n_seqs", _u32), ("max_pages", _u32), ("table", _vp),
                ("len", _vp), ("free_pages", _vp), ("n_free", _vp),
                ("dev", ctypes.c_int)]


class Plan(ctypes.Structure):
    """struct janas_attn_plan."""
    _fields_ = [(x, _vp) for x in ("n_new", "len", "n_free", "granted",
                                   "start", "taken", "slot", "pos", "seq")] + \
        [("max_tokens", _u32)]


class Rows(ctypes.Structure):
    """struct janas_attn_rows."""
    _fields_ = [(x, _vp) for x in ("k", "v", "q", "q_out", "k_norm", "q_norm",
                                   "cs", "sn", "slot", "pos")] + \
        [("eps", ctypes.c_float), ("n_rot", _u32), ("n_tab", _u32),
         ("v_norm", ctypes.c_int), ("n", _u32), ("n_head", _u32),
         ("k_stride", _u32), ("v_stride", _u32), ("q_stride", _u32)]


class PagesCall(ctypes.Structure):
    """struct janas_attn_pages_call."""
    _fields_ = [("q", _vp), ("out", _vp), ("gate", _vp), ("row", _vp),
                ("granted", _vp), ("n_rows", _u32), ("q_stride", _u32),
                ("sel", _vp), ("n_sel", _u32), ("work", _vp),
                ("work_bytes", ctypes.c_size_t), ("out_q8k", _vp)]


class AttnError(RuntimeError):
    def __init__(self, code, what):
        super().__init__(f"{what}: {ERRORS.get(code, code)}")
        self.code = code


_lib = None


def lib():
    """The C-ABI library, loaded once; raises if it was not built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build it with "
                          "`python -m janas_amd.build` (there is no CPU "
                          "fallback)")
    L = ctypes.CDLL(LIB_PATH)
    L.janas_attn_part_bytes.argtypes = [_u32, _u32, _u32, _u32]
    L.janas_attn_part_bytes.restype = ctypes.c_size_t
    L.janas_attn_create.argtypes = [_u32, _u32, _u32, _u32, ctypes.c_int,
                                    ctypes.c_int]
    L.janas_attn_create.restype = _vp
    L.janas_attn_destroy.argtypes = [_vp]
    L.janas_attn_destroy.restype = None
    L.janas_attn_set_scale.argtypes = [_vp, ctypes.c_float]
    L.janas_attn_set_window.argtypes = [_vp, _u32]
    L.janas_attn_set_kv16.argtypes = [_vp, ctypes.c_int]
    L.janas_attn_set_ring.argtypes = [_vp, ctypes.c_int]
    L.janas_attn_ring_positions.argtypes = [_u32, _u32]
    L.janas_attn_ring_positions.restype = _u32
    L.janas_attn_set_last.argtypes = [_vp, _vp]
    L.janas_attn_scores_mode.argtypes = [_vp]
    L.janas_attn_scores_mode.restype = ctypes.c_int
    L.janas_attn_scores_auto.argtypes = [_vp]
    L.janas_attn_scores_auto.restype = ctypes.c_int
    L.janas_attn_run.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _u32,
                                 _u32, _vp]
    L.janas_attn_run.restype = None
    for name in ("janas_attn_run_dev", "janas_attn_run_dev_split",
                 "janas_attn_run_dev_prefill", "janas_attn_run_dev_noalloc"):
        f = getattr(L, name)
        f.argtypes = [_vp, ctypes.c_int, ctypes.c_int, ctypes.POINTER(Seq),
                      _u32, _vp]
        f.restype = ctypes.c_int
    L.janas_attn_run_dev_kernels.argtypes = [_vp, ctypes.c_int, ctypes.c_int,
                                             ctypes.POINTER(Seq), _u32, _vp,
                                             ctypes.c_int]
    L.janas_attn_run_dev_kernels.restype = ctypes.c_int
    L.janas_attn_status.argtypes = [_vp]
    L.janas_attn_status.restype = ctypes.c_int
    L.janas_attn_clear_status.argtypes = [_vp]
    L.janas_attn_clear_status.restype = None
    L.janas_attn_set_abort.argtypes = [_vp, ctypes.c_int]
    L.janas_attn_set_abort.restype = None
    L.janas_attn_import.argtypes = [_vp, _vp, ctypes.c_size_t]
    L.janas_attn_import.restype = ctypes.c_int
    L.janas_attn_sync.argtypes = [_vp, _vp, ctypes.c_size_t, ctypes.c_int]
    L.janas_attn_sync.restype = ctypes.c_int
    L.janas_attn_forget.argtypes = [_vp, _vp]
    L.janas_attn_forget.restype = None
    L.janas_attn_strerror.argtypes = [ctypes.c_int]
    L.janas_attn_strerror.restype = ctypes.c_char_p
    L.janas_attn_cache_write.argtypes = [ctypes.POINTER(Cache), _vp, _vp,
                                         _vp, ctypes.c_float, _vp, _vp, _u32,
                                         ctypes.c_int, _u32, _u32, _vp]
    L.janas_attn_cache_write.restype = ctypes.c_int
    L.janas_attn_q_prep.argtypes = [_vp, _vp, ctypes.c_float, _vp, _vp, _u32,
                                    _u32, _u32, _u32, _vp]
    L.janas_attn_q_prep.restype = ctypes.c_int
    L.janas_attn_cache_shift.argtypes = [ctypes.POINTER(Cache), _u32, _u32,
                                         _u32, _vp, _vp, _u32, _vp]
    L.janas_attn_cache_shift.restype = ctypes.c_int
    L.janas_attn_cache_copy.argtypes = [ctypes.POINTER(Cache), _u32, _u32,
                                        _vp, _vp, _vp, _vp, ctypes.c_int, _vp]
    L.janas_attn_cache_copy.restype = ctypes.c_int
    L.janas_attn_pages_plan.argtypes = [ctypes.POINTER(Pages),
                                        ctypes.POINTER(Plan), _vp]
    L.janas_attn_pages_write.argtypes = [ctypes.POINTER(Pages),
                                         ctypes.POINTER(Rows), _vp]
    L.janas_attn_pages_bounds.argtypes = [ctypes.POINTER(Pages), _vp, _u32, _vp]
    L.janas_attn_pages_work_bytes.argtypes = [_vp, ctypes.POINTER(Pages)]
    L.janas_attn_pages_work_bytes.restype = ctypes.c_size_t
    L.janas_attn_pages_run.argtypes = [_vp, ctypes.POINTER(Pages), ctypes.c_int,
                                       ctypes.POINTER(PagesCall), _vp]
    L.janas_attn_pages_select.argtypes = [_vp, ctypes.POINTER(Pages),
                                          ctypes.POINTER(PagesCall), _u32, _u32,
                                          _vp, _vp]
    for name in ("plan", "write", "bounds", "run", "select"):
        getattr(L, "janas_attn_pages_" + name).restype = ctypes.c_int
    L.janas_attn_prof_enable.argtypes = [_vp, ctypes.c_int]
    L.janas_attn_prof_read.argtypes = [_vp, ctypes.POINTER(_u32),
                                       ctypes.POINTER(ctypes.c_double)]
    L.janas_attn_prof_read.restype = ctypes.c_int
    _lib = L
    return L


def header_functions():
    """The function names include/janas_attn.h declares."""
    text = open(HEADER).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(janas_attn_\w+)\s*\(", text)))


def ptr(x):
    """Address of a numpy array, a torch tensor or an int; None for None."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    return x.ctypes.data


def part_bytes(n_head, n_kv, head_dim, n_ctx):
    return lib().janas_attn_part_bytes(n_head, n_kv, head_dim, n_ctx)


def ring_positions(window, n):
    return lib().janas_attn_ring_positions(window, n)


def strerror(code):
    return lib().janas_attn_strerror(code).decode()


class Attention:
    """One attention instance: janas_attn_create(n_head, n_head_kv,
    head_dim, n_ctx, n_threads, scores)."""

    def __init__(self, n_head, n_kv, head_dim, n_ctx, threads=1,
                 scores=AUTO):
        self._a = lib().janas_attn_create(n_head, n_kv, head_dim, n_ctx,
                                          threads, scores)
        if not self._a:
            raise ValueError("janas_attn_create refused "
                             f"{n_head}/{n_kv}/{head_dim}/{n_ctx}")
        self.n_head, self.n_kv, self.hd, self.n_ctx = (n_head, n_kv,
                                                       head_dim, n_ctx)
        self._last = None

    def close(self):
        if self._a:
            lib().janas_attn_destroy(self._a)
            self._a = None

    destroy = close

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_scale(self, scale):
        lib().janas_attn_set_scale(self._a, scale)

    def set_window(self, window):
        lib().janas_attn_set_window(self._a, window)

    def set_kv16(self, on):
        lib().janas_attn_set_kv16(self._a, 1 if on else 0)

    def set_ring(self, on):
        lib().janas_attn_set_ring(self._a, 1 if on else 0)

    def set_last(self, last):
        """last: a host uint32 array kept alive until the next run."""
        self._last = last
        lib().janas_attn_set_last(self._a, ptr(last))

    def scores_mode(self):
        return lib().janas_attn_scores_mode(self._a)

    def scores_auto(self):
        return lib().janas_attn_scores_auto(self._a)

    def run(self, q, k, ks, v, vs, n, pos0, out):
        """janas_attn_run: synchronous; numpy (host) or device arrays."""
        lib().janas_attn_run(self._a, None, ptr(q), ptr(k), ptr(ks), ptr(v),
                             ptr(vs), n, pos0, ptr(out))
        self._last = None

    def status(self):
        """janas_attn_status: the first device failure kept, or 0."""
        return lib().janas_attn_status(self._a)

    def clear_status(self):
        lib().janas_attn_clear_status(self._a)

    def set_abort(self, on):
        """janas_attn_set_abort: whether janas_attn_run aborts on a
        failure (the default) or returns with a NaN output."""
        lib().janas_attn_set_abort(self._a, 1 if on else 0)

    def import_host(self, arr):
        """janas_attn_import of a host numpy array's bytes (the array
        must stay alive while imported): 0 or a JANAS_ATTN_E* code."""
        return lib().janas_attn_import(self._a, ptr(arr), arr.nbytes)

    def sync(self, arr, to_device=True):
        """janas_attn_sync of a host array (or a view into an imported
        one)."""
        return lib().janas_attn_sync(self._a, ptr(arr), arr.nbytes,
                                     1 if to_device else 0)

    def forget(self, arr):
        """janas_attn_forget of the import holding arr's first byte."""
        lib().janas_attn_forget(self._a, ptr(arr))

    def prepare(self, kv_type, seqs, gate_mode=GATE_NONE, stream=None,
                path="auto"):
        """The call janas_attn_run_dev would make, with its arguments built
        once: returns a function of no arguments that makes it (the arrays
        must stay alive). seqs: dicts with k, v, ks, vs, q, out, gate, last
        (device arrays or addresses), cap, n, pos0, last_max."""
        arr = (Seq * len(seqs))()
        for i, s in enumerate(seqs):
            arr[i] = Seq(ptr(s["k"]), ptr(s["v"]), ptr(s.get("ks")),
                         ptr(s.get("vs")), ptr(s["q"]), ptr(s["out"]),
                         ptr(s.get("gate")), ptr(s.get("last")), s["cap"],
                         s["n"], s["pos0"], s.get("last_max", 0),
                         ptr(s.get("out_q8k")))
        a, n, st = self._a, len(seqs), ptr(stream)
        if path in ("split-kernel", "merge-kernel"):
            # one kernel of the split path alone (measurement)
            kern = 1 if path == "split-kernel" else 2
            f = lib().janas_attn_run_dev_kernels

            def fn(a_, kv_, g_, arr_, n_, st_):
                return f(a_, kv_, g_, arr_, n_, st_, kern)
        else:
            fn = {"auto": lib().janas_attn_run_dev,
                  "split": lib().janas_attn_run_dev_split,
                  "prefill": lib().janas_attn_run_dev_prefill,
                  "noalloc": lib().janas_attn_run_dev_noalloc}[path]

        def call():
            rc = fn(a, kv_type, gate_mode, arr, n, st)
            if rc != 0:
                raise AttnError(rc, f"janas_attn_run_dev ({path})")
        call.keep = (arr, seqs)
        return call

    def run_dev(self, kv_type, seqs, gate_mode=GATE_NONE, stream=None,
                path="auto"):
        """janas_attn_run_dev over a list of sequences (see prepare)."""
        self.prepare(kv_type, seqs, gate_mode, stream, path)()

    # ---- Part 4: single tokens over a paged cache ----

    def pages_work_bytes(self, p):
        """janas_attn_pages_work_bytes: device bytes of `work` for calls over
        the pool p (0 where they would be refused)."""
        return lib().janas_attn_pages_work_bytes(self._a, ctypes.byref(p))

    def _pages_call(self, p, q, out, gate, sel, n_sel, rows, granted, work,
                    out_q8k, gate_mode=GATE_NONE):
        """struct janas_attn_pages_call of tensors q (rows, n_head, hd)."""
        if (rows is None) != (granted is None):
            raise ValueError("rows and granted: both or neither")
        n, shape = q.shape[0], (q.shape[0], self.n_head, self.hd)
        if rows is None and n != p.n_seqs:
            raise ValueError(f"q has {n} rows, the pool {p.n_seqs} sequences")
        stride = _rows_of(q, "q", shape)
        _dense(out, "out", "float32", shape)
        if gate is not None:
            _dense(gate, "gate", "float32",
                   shape[:2] if gate_mode == GATE_HEAD else shape)
        _dense(sel, "sel", "int32", (p.n_seqs, p.n_kv, n_sel))
        # (a step's start has an entry behind the last sequence)
        _dense(rows, "rows", "int32", least=p.n_seqs)
        _dense(granted, "granted", "int32", least=p.n_seqs)
        _dense(work, "work")
        if out_q8k is not None:
            _dense(out_q8k, "out_q8k", "uint8",
                   least=n * (self.n_head * self.hd // 256) * Q8K_BYTES)
        return PagesCall(ptr(q), ptr(out), ptr(gate), ptr(rows), ptr(granted),
                         n, stride, ptr(sel), n_sel, ptr(work),
                         work.numel() * work.element_size(), ptr(out_q8k))

    def prepare_pages(self, p, q, out, *, work, gate=None, gate_mode=GATE_NONE,
                      sel=None, rows=None, granted=None, out_q8k=None,
                      stream=None):
        """The call of janas_attn_pages_run with its arguments built once:
        returns a function of no arguments that makes it (the tensors must
        stay alive). q (a row may be strided), out, gate: device floats
        (sequences or, with rows and granted, packed rows, n_head, hd); sel:
        int32 (n_seqs, n_kv, n_sel) or None."""
        n_sel = 0 if sel is None else sel.shape[2]
        c = self._pages_call(p, q, out, gate, sel, n_sel, rows, granted, work,
                             out_q8k, gate_mode)
        return _prepared("janas_attn_pages_run", self._a, ctypes.byref(p),
                         gate_mode, ctypes.byref(c), ptr(stream),
                         keep=(p, c, self, q, out, gate, sel, rows, granted,
                               work, out_q8k))

    def run_pages(self, p, q, out, **more):
        """janas_attn_pages_run (see prepare_pages)."""
        self.prepare_pages(p, q, out, **more)()

    def prepare_select(self, p, q, sel, *, work, first=1, last=1, rows=None,
                       granted=None, stream=None):
        """The call of janas_attn_pages_select, as prepare_pages: blocks into
        sel, int32 (n_seqs, n_kv, n_sel)."""
        c = self._pages_call(p, q, None, None, sel, sel.shape[2], rows, granted,
                             work, None)
        return _prepared("janas_attn_pages_select", self._a, ctypes.byref(p),
                         ctypes.byref(c), first, last, ptr(sel), ptr(stream),
                         keep=(p, c, self, q, sel, rows, granted, work))

    def select(self, p, q, sel, **more):
        """janas_attn_pages_select (see prepare_select)."""
        self.prepare_select(p, q, sel, **more)()

    def prof_enable(self, on=True):
        lib().janas_attn_prof_enable(self._a, 1 if on else 0)

    def prof_read(self):
        """{kernel: (launches, ms)} for split, merge and prefill."""
        counts = (_u32 * 3)()
        ms = (ctypes.c_double * 3)()
        rc = lib().janas_attn_prof_read(self._a, counts, ms)
        if rc != 0:
            raise AttnError(rc, "janas_attn_prof_read")
        return {name: (counts[i], ms[i])
                for i, name in enumerate(("split", "merge", "prefill"))}


# ---- Part 3: the cache around the attention --------------------------------

def _check(rc, what):
    if rc != 0:
        raise AttnError(rc, what)


def cache(k, v, ks=None, vs=None, *, kv_type, ring=False):
    """struct janas_attn_cache over device tensors k, v (n_kv, cap, hd) and
    ks, vs (n_kv, cap)."""
    n_kv, cap, hd = k.shape
    return Cache(ptr(k), ptr(v), ptr(ks), ptr(vs), n_kv, hd, cap, kv_type,
                 1 if ring else 0)


def cache_write(c, k, v, *, cs, sn, n_rot, pos0, k_norm=None, eps=1e-6,
                v_norm=False, stream=None):
    """janas_attn_cache_write: k, v (n, n_kv, hd) device floats."""
    _check(lib().janas_attn_cache_write(ctypes.byref(c), ptr(k), ptr(v),
                                        ptr(k_norm), eps, ptr(cs), ptr(sn),
                                        n_rot, 1 if v_norm else 0, pos0,
                                        k.shape[0], ptr(stream)),
           "janas_attn_cache_write")


def q_prep(q, *, cs, sn, n_rot, q_norm=None, eps=1e-6, stream=None):
    """janas_attn_q_prep on q (n, n_head, hd), in place."""
    n, n_head, hd = q.shape
    _check(lib().janas_attn_q_prep(ptr(q), ptr(q_norm), eps, ptr(cs), ptr(sn),
                                   n_rot, n, n_head, hd, ptr(stream)),
           "janas_attn_q_prep")


def cache_shift(c, *, keep, drop, n_pos, cs, sn, n_rot, stream=None):
    """janas_attn_cache_shift."""
    _check(lib().janas_attn_cache_shift(ctypes.byref(c), keep, drop, n_pos,
                                        ptr(cs), ptr(sn), n_rot, ptr(stream)),
           "janas_attn_cache_shift")


def cache_copy(c, *, n_pos, rows, k, v, ks=None, vs=None, out=True,
               stream=None):
    """janas_attn_cache_copy: out=True cache -> buffers, else back."""
    _check(lib().janas_attn_cache_copy(ctypes.byref(c), n_pos, rows, ptr(k),
                                       ptr(v), ptr(ks), ptr(vs),
                                       1 if out else 0, ptr(stream)),
           "janas_attn_cache_copy")


# ---- Part 4: a paged cache --------------------------------------------------

_KV_NAME = {KV_I8: "int8", KV_I16: "int16", KV_F16: "float16",
            KV_F32: "float32"}


def _dense(x, what, dtype=None, shape=None, least=None):
    """x (a torch tensor, or None) as an entry point reads it: packed, of this
    type and shape, of `least` elements at least."""
    if x is None:
        return
    if not x.is_contiguous():
        raise ValueError(f"{what} is not contiguous")
    if dtype and str(x.dtype) != "torch." + dtype:
        raise ValueError(f"{what} is {x.dtype}, not {dtype}")
    if shape and tuple(x.shape) != tuple(shape):
        raise ValueError(f"{what} is {tuple(x.shape)}, not {tuple(shape)}")
    if least is not None and x.numel() < least:
        raise ValueError(f"{what} has {x.numel()} elements, not {least}")


def _rows_of(x, what, shape):
    """Rows (n, heads, hd) of floats, each row packed: the floats from one row
    to the next."""
    if str(x.dtype) != "torch.float32":
        raise ValueError(f"{what} is {x.dtype}, not float32")
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{what} is {tuple(x.shape)}, not {tuple(shape)}")
    _dense(x[0] if x.shape[0] else x, what + "'s rows")
    if x.shape[0] < 2:
        return 0
    if x.stride(0) < shape[1] * shape[2]:
        raise ValueError(f"{what}'s rows overlap")
    if x.stride(0) > 0xFFFFFFFF:
        raise ValueError(f"{what}'s rows are {x.stride(0)} floats apart, more than 32 bits hold")
    return x.stride(0)


def _prepared(name, *args, keep):
    """A call of an entry point as a function of no arguments. The tensors among
    what it keeps and its pool (keep[0]) are on one GPU."""
    f = getattr(lib(), name)
    where = {str(x.device) for x in keep + keep[0].keep if hasattr(x, "device")}
    if len(where) > 1:
        raise ValueError(f"{name}: tensors on {', '.join(sorted(where))}")
    host = not any(x.startswith("cuda") for x in where)

    def call():
        if host:
            raise ValueError(f"{name}: tensors in host memory")
        rc = f(*args)
        if rc != 0:
            raise AttnError(rc, name)
    call.keep = keep
    return call


def page_tables(table, length, *, page, free=None, n_free=None, n_pages=None):
    """struct janas_attn_pages with the sequences' half alone, for
    pages_plan: table int32 (n_seqs, max_pages), length int32 (n_seqs), free
    int32 (n_pages), n_free int32 (1)."""
    _dense(table, "table", "int32")
    n_seqs, max_pages = table.shape
    _dense(length, "length", "int32", (n_seqs,))
    _dense(free, "free", "int32", None if n_pages is None else (n_pages,))
    _dense(n_free, "n_free", "int32", (1,))
    if n_pages is None:
        n_pages = 0 if free is None else free.shape[0]
    p = Pages(n_pages=n_pages, page=page, n_seqs=n_seqs, max_pages=max_pages,
              table=ptr(table), len=ptr(length), free_pages=ptr(free),
              n_free=ptr(n_free), dev=table.device.index or 0)
    p.keep = (table, length, free, n_free)
    return p


def pages(k, v, ks=None, vs=None, *, kv_type, table, length, free=None,
          n_free=None, bounds=None):
    """struct janas_attn_pages over device tensors k, v (n_pages, n_kv, page,
    hd), ks, vs (n_pages, n_kv, page), bounds float16 (n_pages, n_kv, 2, hd)
    and page_tables' (kept alive by it)."""
    n_pages, n_kv, page, hd = k.shape
    for x, what in ((k, "k"), (v, "v")):
        _dense(x, what, _KV_NAME[kv_type], (n_pages, n_kv, page, hd))
    for x, what in ((ks, "ks"), (vs, "vs")):
        _dense(x, what, "float32", (n_pages, n_kv, page))
    _dense(bounds, "bounds", "float16", (n_pages, n_kv, 2, hd))
    p = page_tables(table, length, page=page, free=free, n_free=n_free,
                    n_pages=n_pages)
    p.k, p.v, p.ks, p.vs, p.bounds = ptr(k), ptr(v), ptr(ks), ptr(vs), ptr(bounds)
    p.n_kv, p.head_dim, p.kv_type = n_kv, hd, kv_type
    p.dev = k.device.index or 0
    p.keep += (k, v, ks, vs, bounds)
    return p


def prepare_pages_plan(p, n_new, *, slot, pos, seq, start, taken, granted,
                       length, n_free, stream=None):
    """The call of janas_attn_pages_plan with its arguments built once:
    returns a function of no arguments that makes it. n_new int32 (n_seqs), -1:
    release; length, n_free: where the new ones go (the pool's own tensors, or
    others); slot, pos, seq: int32 of as many rows as the step may have."""
    n = p.n_seqs
    for x, what, m in ((n_new, "n_new", n), (length, "length", n),
                       (granted, "granted", n), (n_free, "n_free", 1),
                       (start, "start", n + 1), (taken, "taken", n + 1)):
        _dense(x, what, "int32", (m,))
    for x, what in ((slot, "slot"), (pos, "pos"), (seq, "seq")):
        _dense(x, what, "int32", slot.shape)
    s = Plan(ptr(n_new), ptr(length), ptr(n_free), ptr(granted), ptr(start),
             ptr(taken), ptr(slot), ptr(pos), ptr(seq), slot.numel())
    return _prepared("janas_attn_pages_plan", ctypes.byref(p), ctypes.byref(s),
                     ptr(stream), keep=(p, s, n_new, length, n_free, granted,
                                        start, taken, slot, pos, seq))


def pages_plan(p, n_new, **more):
    """janas_attn_pages_plan (see prepare_pages_plan)."""
    prepare_pages_plan(p, n_new, **more)()


def prepare_pages_write(p, k, v, *, slot, pos=None, cs=None, sn=None, n_rot=0,
                        k_norm=None, eps=1e-6, v_norm=False, q=None,
                        q_out=None, q_norm=None, stream=None):
    """The call of janas_attn_pages_write, as prepare_pages_plan. k, v (n,
    n_kv, hd) and q (n, n_head, hd): device floats whose rows may be strided;
    q_out: packed (q itself if None); cs, sn (positions, n_rot / 2)."""
    n, n_head = k.shape[0], 0
    strides = [_rows_of(x, what, (n, p.n_kv, p.head_dim))
               for x, what in ((k, "k"), (v, "v"))] + [0]
    if q is not None:
        n_head = q.shape[1]
        strides[2] = _rows_of(q, "q", (n, n_head, p.head_dim))
        q_out = q if q_out is None else q_out
        _dense(q_out, "q_out", "float32", q.shape)
    for x, what in ((slot, "slot"), (pos, "pos")):
        _dense(x, what, "int32", (n,))
    n_tab = 0
    if n_rot:
        n_tab = cs.shape[0]
        for x, what in ((cs, "cs"), (sn, "sn")):
            _dense(x, what, "float32", (n_tab, n_rot // 2))
    for x, what in ((k_norm, "k_norm"), (q_norm, "q_norm")):
        _dense(x, what, "float32", (p.head_dim,))
    r = Rows(ptr(k), ptr(v), ptr(q), ptr(q_out), ptr(k_norm), ptr(q_norm),
             ptr(cs), ptr(sn), ptr(slot), ptr(pos), eps, n_rot, n_tab,
             1 if v_norm else 0, n, n_head, *strides)
    return _prepared("janas_attn_pages_write", ctypes.byref(p), ctypes.byref(r),
                     ptr(stream), keep=(p, r, k, v, q, q_out, k_norm, q_norm,
                                        cs, sn, slot, pos))


def pages_write(p, k, v, **more):
    """janas_attn_pages_write (see prepare_pages_write)."""
    prepare_pages_write(p, k, v, **more)()


def prepare_pages_bounds(p, n_new=None, *, max_new=0, stream=None):
    """The call of janas_attn_pages_bounds, as prepare_pages_plan: n_new int32
    (n_seqs), or None: all blocks."""
    _dense(n_new, "n_new", "int32", (p.n_seqs,))
    return _prepared("janas_attn_pages_bounds", ctypes.byref(p), ptr(n_new),
                     max_new, ptr(stream), keep=(p, n_new))


def pages_bounds(p, n_new=None, **more):
    """janas_attn_pages_bounds (see prepare_pages_bounds)."""
    prepare_pages_bounds(p, n_new, **more)()
