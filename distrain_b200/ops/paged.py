"""Paged key/value cache of the serving path: page tables, the append of new rows, attention over pages.

The cache of one layer is two tensors ``[pages, nkv, page_size, d]`` bf16 (K after the position rotation, V).
A request's *table row* lists its pages in order; the *slot* of a token is ``page * page_size + offset``.
One step of a batch, all on the GPU and fit for capture in a CUDA graph (every buffer is the caller's):

    page_tables(...)        lengths -> new table entries, slot and position of every new token
    plan.build(...)         lengths -> the work list of the step's attention, shared by all layers
    per layer: kv_append(...) bias + rotation of the QKV rows, K and V into their slots
               paged_attention(...) queries over the pages, shared prefixes computed once for their group

Calls check types, shapes and devices and raise ``ValueError``. What only the GPU can see is reported through
``ops.device_error`` and touches no other request: the append leaves out a row whose slot or position is none, the
attention takes keys and values on a page outside the cache as zeros (their request's rows are then meaningless), and
lengths that contradict each other leave the step without work. Such a report stays until ``ops.clear_device_error``;
it stops no other call.

A decode step's calls take a few microseconds on the GPU, so what they cost here counts: each call tests its
arguments in one expression and only names what is wrong once that has failed, and the launchers take one packed
struct.
"""
from __future__ import annotations

import struct

import torch

from ._lib import LAUNCHES, lib, check, register, c_int, c_ll, c_void

PAGE_SIZES = (16, 32, 64, 128)
MAX_REQUESTS = 8192
MAX_GROUP_HEADS = 16
POOL_EMPTY, TABLE_FULL, SLOTS_FULL, NEGATIVE_LENGTH = 1, 2, 4, 8  # bits of page_tables' used[1]

_SHIFT = {p: p.bit_length() - 1 for p in PAGE_SIZES}
_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16
# argument structs of the launchers (csrc/kernels/paged.cu, paged_attention.cu)
_TABLES = struct.Struct("=10Qq6i").pack
_APPEND = struct.Struct("=9Qq8i").pack
_PLAN = struct.Struct("=5Q10i").pack
_ATTENTION = struct.Struct("=11Q2qd10i").pack

_fns = {}


def _fn(name):
    """The launcher ``name`` (its signature is declared on first use)."""
    f = _fns.get(name)
    if f is None:
        import ctypes
        if name.endswith("bytes"):
            f = register(name, [c_int] * 6, restype=c_ll)
        elif name == "dt_paged_kernels":
            f = register(name, [c_int] * 6)
        else:
            f = register(name, [ctypes.c_char_p, c_void])
        _fns[name] = f
    return f


def _fail(msg):
    raise ValueError(msg)


def _launch(name, args, stream):
    """Calls a launcher, which sees for itself what depends on addresses."""
    rc = (_fns.get(name) or _fn(name))(args, stream)
    if rc == 0:
        LAUNCHES[0] += 1
        return
    if rc == -13:
        _fail(f"{name[3:]}: outputs must not share memory with inputs or each other")
    if rc == -11:
        _fail(f"{name[3:]}: rows and tables of floats must start on a 16-byte boundary")
    check(rc, name)


def _vec(name, t, n, dtype=_I32):
    """A contiguous vector of ``n`` elements (any number when None)."""
    if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
        _fail(f"{name}: expected a contiguous {dtype} vector" + (f" of {n}" if n is not None else "") +
              f", got {t.dtype} {tuple(t.shape)}")


def _rows(name, t, shape, dtype=_BF16):
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        _fail(f"{name}: expected contiguous {dtype} {shape}, got {t.dtype} {tuple(t.shape)}")


def _table(name, t, rows):
    if t.dtype != _I32 or t.dim() != 2 or t.shape[0] != rows or \
            (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        _fail(f"{name}: expected int32 rows [{rows}, width] with unit column stride, got {t.dtype} {tuple(t.shape)}")


_current = torch._C._cuda_getDevice


def on_current_device(*tensors):
    """The current device, which all ``tensors`` (None skipped) must live on: kernels launch there."""
    for t in tensors:
        if t is not None:
            if not t.is_cuda:
                _fail("expected CUDA tensors")
            if t.get_device() != _current():
                _fail(f"tensor on {t.device}, but the current device is cuda:{_current()}")
    return _current()


def _stream(stream, dev):
    return torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream


def _page_shift(page_size):
    shift = _SHIFT.get(page_size)
    return _fail(f"page_size {page_size}: one of {PAGE_SIZES}") if shift is None else shift


def page_tables(cached, new, free, tables, slots, positions, cu, total, used, *, page_size, start=None, stream=None):
    """Pages for the new tokens of every request, and where each new token goes.

    Request i has ``cached[i]`` tokens in the pages of table row i and adds ``new[i]`` (int32 [B]). The pages it
    needs are taken in request order from the front of ``free`` (int32 page ids) and written behind its
    ``ceil(cached / page_size)`` present entries of ``tables`` ([B, width] int32, written in place).
    Outputs: ``cu`` [B+1] running sums of ``new``; ``total`` [B] = cached + new; for token ``cu[i] + j`` its
    ``slots`` entry and ``positions`` entry ``start[i] + cached[i] + j`` (``start`` [B], 0 when None: the length
    of a shared prefix). ``slots`` may hold more than the step's tokens (a captured graph's capacity): those
    behind get slot -1, which ``kv_append`` skips, those on a page id that is negative or too large for an int32 slot
    get 2^31 - 1, which it reports. ``used`` [2] = pages taken, and why nothing was: 0, or a sum
    of POOL_EMPTY, TABLE_FULL (a request of about 2^31 tokens too), SLOTS_FULL, NEGATIVE_LENGTH - then the table is
    untouched, every slot is -1, ``cu`` is zero and ``total`` equals ``cached``. Outputs must not share memory with
    inputs or each other."""
    shift = _SHIFT.get(page_size)
    rows, n = cached.shape, slots.shape
    B, ts = rows[0] if len(rows) == 1 else 0, tables.shape
    if not (shift is not None and 0 < B <= MAX_REQUESTS and len(ts) == 2 and ts[0] == B and tables.is_contiguous() and
            len(n) == 1 and n[0] <= 1 << 30 and new.shape == rows and total.shape == rows and positions.shape == n and
            cu.shape == (B + 1,) and used.shape == (2,) and free.dim() == 1 and
            cached.dtype is _I32 and new.dtype is _I32 and free.dtype is _I32 and tables.dtype is _I32 and
            slots.dtype is _I32 and positions.dtype is _I32 and cu.dtype is _I32 and total.dtype is _I32 and
            used.dtype is _I32 and cached.is_contiguous() and new.is_contiguous() and free.is_contiguous() and
            slots.is_contiguous() and positions.is_contiguous() and cu.is_contiguous() and total.is_contiguous() and
            used.is_contiguous()):
        shift = _page_shift(page_size)
        if len(rows) != 1 or not 1 <= B <= MAX_REQUESTS:
            _fail(f"cached: 1 to {MAX_REQUESTS} requests, got {tuple(rows)}")
        _vec("cached", cached, B)
        _vec("new", new, B)
        _vec("free", free, None)
        _table("tables", tables, B)
        _vec("slots", slots, None)
        _vec("positions", positions, n[0])
        _vec("cu", cu, B + 1)
        _vec("total", total, B)
        _vec("used", used, 2)
        if n[0] > 1 << 30:
            _fail("slots: at most 2^30 tokens")
    if start is not None:
        _vec("start", start, B)
    n_free = free.shape[0]
    if n_free >= 1 << 31:
        _fail("free: below 2^31 pages")
    a, b, f, s = cached.data_ptr(), new.data_ptr(), free.data_ptr(), 0 if start is None else start.data_ptr()
    o = (tables.data_ptr(), slots.data_ptr(), positions.data_ptr(), cu.data_ptr(), total.data_ptr(), used.data_ptr())
    dev = cached.get_device()
    if not (dev >= 0 and new.get_device() == dev and free.get_device() == dev and tables.get_device() == dev and
            slots.get_device() == dev and positions.get_device() == dev and cu.get_device() == dev and
            total.get_device() == dev and used.get_device() == dev and (start is None or start.get_device() == dev) and
            _current() == dev):
        out = [p for p in o if p]  # (the launcher looks at every byte, but tensors that are not on a GPU do not get there)
        if len(set(out)) < len(out) or {a, b, f, s} & set(out):
            _fail("outputs must not share memory with inputs or each other")
        on_current_device(cached, new, free, tables, slots, positions, cu, total, used, start)
    _launch("dt_page_tables", _TABLES(a, b, s, f, *o, tables.stride(0), n_free, ts[1], n[0], B, shift, 0),
            _stream(stream, dev))


def _cache(k_cache, v_cache):
    """(pages, nkv, page_size, d) of a layer's cache."""
    shape = k_cache.shape
    if not (len(shape) == 4 and v_cache.shape == shape and k_cache.dtype is _BF16 and v_cache.dtype is _BF16 and
            k_cache.is_contiguous() and v_cache.is_contiguous() and shape[2] in _SHIFT and
            0 < shape[0] * shape[1] * shape[2] < 1 << 31):
        if len(shape) != 4:
            _fail(f"k_cache: expected [pages, nkv, page_size, d], got {tuple(shape)}")
        _rows("k_cache", k_cache, tuple(shape))
        _rows("v_cache", v_cache, tuple(shape))
        _page_shift(shape[2])
        _fail("cache: at least one page and below 2^31 rows (pages * nkv * page_size)")
    return shape


def kv_append(qkv, bias, cos, sin, slots, positions, q, k_cache, v_cache, *, stream=None):
    """Bias and rotary embedding of the step's QKV rows, K and V written to their slots.

    ``qkv`` [T, (nh + 2 nkv) d] bf16 (rows may be strided: the QKV GEMM's output without bias), ``bias`` fp32
    or None, ``cos`` / ``sin`` [max_pos, d/2] fp32 tables of the rotate-half form. Row t with slot ``slots[t]``
    >= 0: ``q[t]`` = rot(q + bias), K row = rot(k + bias), V row = v + bias, each rounded once to bf16; a row
    with a negative slot is left out (its ``q`` row too). Two rows of one call must not have the same slot, and
    ``q``, ``k_cache`` and ``v_cache`` must not share memory with each other or an input.
    A slot outside the cache or a position outside the tables leaves its row out and is reported."""
    pages, nkv, page_size, d = _cache(k_cache, v_cache)
    rows, qs, cs = qkv.shape, q.shape, cos.shape
    if d % 16 or d < 16:
        _fail(f"head dim {d}: a multiple of 16")
    if len(rows) != 2 or len(qs) != 2 or qs[1] % d or qs[1] == 0:
        _fail(f"q: [tokens, nh * d] with d = {d}, got {tuple(qs)}; qkv: two-dimensional")
    T, nh = rows[0], qs[1] // d
    W = qs[1] + 2 * nkv * d
    ld, one = qkv.stride()
    if T <= 1:
        ld = W
    if not (rows[1] == W and qkv.dtype is _BF16 and one == 1 and ld >= W and ld % 8 == 0 and qs[0] == T and
            q.dtype is _BF16 and q.is_contiguous() and slots.shape == (T,) and positions.shape == (T,) and
            slots.dtype is _I32 and positions.dtype is _I32 and slots.is_contiguous() and positions.is_contiguous() and
            len(cs) == 2 and cs[0] > 0 and cs[1] == d // 2 and sin.shape == cs and cos.dtype is _F32 and
            sin.dtype is _F32 and cos.is_contiguous() and sin.is_contiguous()):
        if qkv.dtype != _BF16 or rows[1] != W or one != 1 or ld < W or ld % 8:
            _fail(f"qkv: bf16 [T, {W}] rows with a stride of a multiple of 8, got {qkv.dtype} {tuple(rows)} strides "
                  f"{qkv.stride()}")
        _rows("q", q, (T, nh * d))
        _vec("slots", slots, T)
        _vec("positions", positions, T)
        if len(cs) != 2 or cs[0] < 1:
            _fail(f"cos: [max_pos, {d // 2}], got {tuple(cs)}")
        _rows("cos", cos, (cs[0], d // 2), _F32)
        _rows("sin", sin, tuple(cs), _F32)
    if bias is not None:
        _vec("bias", bias, W, _F32)
    dev = qkv.get_device()
    if not (dev >= 0 and (bias is None or bias.get_device() == dev) and cos.get_device() == dev and
            sin.get_device() == dev and slots.get_device() == dev and positions.get_device() == dev and
            q.get_device() == dev and k_cache.get_device() == dev and v_cache.get_device() == dev and _current() == dev):
        on_current_device(qkv, bias, cos, sin, slots, positions, q, k_cache, v_cache)
    if T == 0:
        return
    _launch("dt_kv_append", _APPEND(qkv.data_ptr(), 0 if bias is None else bias.data_ptr(), cos.data_ptr(),
                                    sin.data_ptr(), slots.data_ptr(), positions.data_ptr(), q.data_ptr(),
                                    k_cache.data_ptr(), v_cache.data_ptr(), ld, cs[0], T, nh, nkv, d,
                                    _SHIFT[page_size], pages, 0), _stream(stream, dev))


class AttentionPlan:
    """Buffers of the attention of one batch shape: the step's work list and the scratch of its partial results.

    Room for ``tokens`` query rows (the row count of ``q``), ``requests`` and ``groups`` (0: no shared prefixes).
    ``build`` lays the work out on the GPU from the step's lengths, once a step; every layer's
    ``paged_attention`` then uses it. Calls on one plan must run in stream order (one plan per stream; graphs
    that replay at the same time need plans of their own)."""

    def __init__(self, tokens, requests, groups=0, *, nh, nkv, d, page_size, device="cuda"):
        self.T, self.B, self.G = int(tokens), int(requests), int(groups)
        self.nh, self.nkv, self.d = int(nh), int(nkv), int(d)
        self.page_size, self.shift = int(page_size), _page_shift(page_size)
        if self.d not in (16, 32, 64, 128):
            _fail(f"head dim {d}: 16, 32, 64 or 128")
        if self.nkv < 1 or self.nh < self.nkv or self.nh % self.nkv or self.nh // self.nkv > MAX_GROUP_HEADS:
            _fail(f"{nh} query heads on {nkv} kv heads: a whole number of up to {MAX_GROUP_HEADS} a kv head")
        if not 1 <= self.B <= MAX_REQUESTS or not 0 <= self.G <= self.B or not 0 <= self.T <= 1 << 24 or \
                self.T * self.nh >= 1 << 29:
            _fail(f"1 to {MAX_REQUESTS} requests, at most as many groups and 2^24 tokens; got {requests}, {groups}, {tokens}")
        dev = torch.device(device)
        if dev.type != "cuda":
            _fail("device: a CUDA device")
        lib()
        shape = (self.T, self.B, self.G, self.nh, self.nkv, self.d)
        with torch.cuda.device(dev):
            self.kernels = _fn("dt_paged_kernels")(*shape)
            plan_bytes, work_bytes = _fn("dt_paged_plan_bytes")(*shape), _fn("dt_paged_work_bytes")(*shape)
            if plan_bytes < 0 or work_bytes < 0:
                _fail(f"no plan for {shape}")
            self.plan = torch.zeros(plan_bytes // 4, dtype=torch.int32, device=dev)
            self.work = torch.empty(work_bytes, dtype=torch.uint8, device=dev)
        self.cu_q = self.tables = self.prefix = None

    def build(self, cu_q, lens, tables, *, prefix=None, stream=None):
        """Work list of a step. ``cu_q`` int32 [B+1]: request i's query rows are ``cu_q[i] .. cu_q[i+1]`` of q
        (rows behind ``cu_q[B]`` belong to nobody); ``lens`` int32 [B]: its own keys, those of this step
        included; ``tables`` int32 [B, width]: their pages. ``prefix`` = (``prefix_tables`` [G, width],
        ``prefix_lens`` [G], ``cu_group`` [G+1]): group y, requests ``cu_group[y] .. cu_group[y+1]``, has
        ``prefix_lens[y]`` keys in front of every request's own (``cu_group`` covers all requests). The tensors
        must stay unchanged until the step's last ``paged_attention`` has run. Lengths that contradict each
        other or the tables are reported and leave the step without work."""
        B, G = self.B, self.G
        ts = tables.shape
        if not (cu_q.shape == (B + 1,) and lens.shape == (B,) and len(ts) == 2 and ts[0] == B and cu_q.dtype is _I32 and
                lens.dtype is _I32 and tables.dtype is _I32 and cu_q.is_contiguous() and lens.is_contiguous() and
                tables.is_contiguous()):
            _vec("cu_q", cu_q, B + 1)
            _vec("lens", lens, B)
            _table("tables", tables, B)
        if (prefix is None) != (G == 0):
            _fail(f"plan for {G} groups: prefix " + ("given" if prefix is not None else "missing"))
        most, most_prefix = ts[1] * self.page_size, 0
        pl = cg = 0
        if prefix is not None:
            pt, pl, cg = prefix
            _table("prefix_tables", pt, G)
            _vec("prefix_lens", pl, G)
            _vec("cu_group", cg, G + 1)
            most_prefix = pt.shape[1] * self.page_size
        if most >= 1 << 30 or most_prefix >= 1 << 30:
            _fail("table rows: below 2^30 tokens")
        dev = cu_q.get_device()
        if not (dev >= 0 and self.plan.get_device() == dev and lens.get_device() == dev and tables.get_device() == dev and
                _current() == dev and prefix is None):
            dev = on_current_device(cu_q, self.plan, lens, tables, *(prefix or ()))
        if prefix is not None:
            pl, cg = pl.data_ptr(), cg.data_ptr()
        check(_fn("dt_paged_plan")(_PLAN(self.plan.data_ptr(), cu_q.data_ptr(), lens.data_ptr(), cg, pl, self.T, B, G,
                                         self.nh, self.nkv, self.d, self.shift, most, most_prefix, 0),
                                   _stream(stream, dev)), "dt_paged_plan")
        self.cu_q, self.tables, self.prefix = cu_q, tables, prefix


def paged_attention(q, k_cache, v_cache, out, plan, *, scale=None, lse=None, stream=None):
    """Attention of the step's queries over the pages of ``plan`` (``AttentionPlan.build`` first).

    Token j of a request with n query rows and ``lens`` own keys sees its group's whole prefix and its own keys
    0 .. lens - n + j. ``q`` and ``out`` [T, nh * d] bf16, T = the plan's tokens; rows behind ``cu_q[B]`` are
    left as they are. ``scale`` (1e-30 to 1e30; scaled scores stay below 2^30) defaults to d ** -0.5. ``lse`` [T, nh]
    fp32 receives the log-sum-exp of the scaled scores. A token that sees no key gets a zero row (lse -inf). What the
    pages hold behind a request's last key does not matter; a non-finite V row of a *later* token of the same request
    may reach earlier ones. ``out`` and ``lse`` must not share memory with each other or an input."""
    pages, nkv, page_size, d = _cache(k_cache, v_cache)
    if nkv != plan.nkv or page_size != plan.page_size or d != plan.d:
        _fail(f"cache of {nkv} kv heads, pages of {page_size}, head dim {d}; plan for {plan.nkv}, {plan.page_size}, {plan.d}")
    cu_q, tables, prefix = plan.cu_q, plan.tables, plan.prefix
    if cu_q is None:
        _fail("plan.build has not been called")
    T, nh = plan.T, plan.nh
    shape = (T, nh * d)
    if not (q.shape == shape and out.shape == shape and q.dtype is _BF16 and out.dtype is _BF16 and q.is_contiguous() and
            out.is_contiguous()):
        _rows("q", q, shape)
        _rows("out", out, shape)
    qp, op = q.data_ptr(), out.data_ptr()
    if op == qp and T:
        _fail("out must not be q")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:  # (zero or infinite in fp32, a masked score's product with it would be NaN)
        _fail(f"scale {scale}: a number from 1e-30 to 1e30")
    if lse is not None:
        _rows("lse", lse, (T, nh), _F32)
    dev = q.get_device()
    if not (dev >= 0 and k_cache.get_device() == dev and v_cache.get_device() == dev and out.get_device() == dev and
            (lse is None or lse.get_device() == dev) and plan.plan.get_device() == dev and _current() == dev):
        on_current_device(q, k_cache, v_cache, out, lse, plan.plan)
    if T == 0:
        return
    pt, ld_prefix, cg, wp = (0, 0, 0, 0) if prefix is None else \
        (prefix[0].data_ptr(), prefix[0].stride(0), prefix[2].data_ptr(), prefix[0].shape[1])
    _launch("dt_paged_attention", _ATTENTION(qp, k_cache.data_ptr(), v_cache.data_ptr(), op,
                                             0 if lse is None else lse.data_ptr(), plan.plan.data_ptr(),
                                             plan.work.data_ptr(), cu_q.data_ptr(), cg, tables.data_ptr(), pt,
                                             tables.stride(0), ld_prefix, scale, T, plan.B, plan.G, nh, nkv, d,
                                             plan.shift, pages, tables.shape[1], wp), _stream(stream, dev))
    LAUNCHES[0] += plan.kernels - 1
