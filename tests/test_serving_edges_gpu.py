"""Serving operators on the GPU at the edges of what their documentation allows."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _i(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _decode_tables(B, P=16):
    """A step of ``B`` requests that each add a token, every third of them on a new page; checked by arithmetic."""
    from distrain_b200.ops import paged
    cached = [(P if i % 3 == 0 else 1 + i % (P - 1)) for i in range(B)]
    opens = [i for i in range(B) if i % 3 == 0]
    tables = torch.full((B, 2), -1, dtype=torch.int32, device=DEV)
    tables[:, 0] = torch.arange(B, dtype=torch.int32, device=DEV)
    free = torch.arange(B, B + len(opens), dtype=torch.int32, device=DEV)
    slots, pos = torch.full((B,), 99, dtype=torch.int32, device=DEV), torch.full((B,), 99, dtype=torch.int32, device=DEV)
    cu, total, used = _i([99] * (B + 1)), _i([99] * B), _i([99, 99])
    paged.page_tables(_i(cached), _i([1] * B), free, tables, slots, pos, cu, total, used, page_size=P)
    assert used.tolist() == [len(opens), 0] and cu.tolist() == list(range(B + 1))
    assert total.tolist() == [c + 1 for c in cached] and pos.tolist() == cached
    want = [(B + i // 3) * P if i % 3 == 0 else i * P + cached[i] for i in range(B)]
    assert slots.tolist() == want
    assert tables[:, 1].tolist() == [B + i // 3 if i % 3 == 0 else -1 for i in range(B)]


def test_page_tables_of_4096_requests_before_any_larger_call():
    """3 * 4 * 4096 bytes of dynamic shared memory are 48 KB, and the kernel's static part comes on top: the first call
    of a process must not rest on a limit that a larger one has raised."""
    code = "import sys; sys.path[:0] = ['', 'tests']; import test_serving_edges_gpu as t; t._decode_tables(4096); print('passed')"
    p = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "passed" in p.stdout, p.stderr[-2000:]


@pytest.mark.parametrize("B", [4073, 4074, 4096, 4097, 8192, 5000])
def test_page_tables_of_many_requests(B):
    _decode_tables(B)


# ───────────────────────── one caller's bad data ─────────────────────────
def _long_calls():
    """Attention of both kernels and a GEMM, whose waits poll many times: (run, outputs)."""
    from distrain_b200 import ops
    from test_paged_gpu import Batch
    batches = [Batch([1] * 64, [4096 - 37 * i for i in range(64)], 16, 4, 128, 64, seed=3),
               Batch([900, 1, 300], [2000, 3000, 300], 16, 4, 128, 64, seed=4)]
    g = torch.Generator(device=DEV).manual_seed(0)
    a, b = (torch.randn(4096, 4096, generator=g, device=DEV).bfloat16() for _ in range(2))

    def run():
        c = torch.full((4096, 4096), 7.0, device=DEV)
        out = [x.run() for x in batches]
        ops.gemm(a, b, c, M=4096, N=4096, K=4096)
        return out + [c]
    return run


@pytest.mark.parametrize("what", ["slot", "page", "lengths"])
def test_a_report_stops_no_other_call(what):
    """Bad data stays reported until it is cleared; the calls after it (and beside it) give what they gave before."""
    from distrain_b200 import ops
    from distrain_b200.ops import paged
    from test_paged_gpu import Batch
    ops.clear_device_error()
    run = _long_calls()
    want = run()
    assert ops.device_error() == (0, 0)
    if what == "slot":
        d, P = 32, 16
        cos = torch.ones(8, d // 2, device=DEV)
        kc, vc = (torch.zeros(2, 2, P, d, device=DEV).bfloat16() for _ in range(2))
        q = torch.zeros(1, 4 * d, device=DEV).bfloat16()
        paged.kv_append(torch.ones(1, 8 * d, device=DEV).bfloat16(), None, cos, cos, _i([2 * P]), _i([0]), q, kc, vc)
        code = 5
    else:
        b = Batch([1, 1], [50, 20], 4, 2, 64, 16)
        if what == "page":
            b.tables[0, 1] = 10 ** 6
        else:
            b.len_t[1] = 10 ** 6
        b.run()
        code = 5 if what == "page" else 6
    assert ops.device_error()[0] == code
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(want, run()))
    assert ops.device_error()[0] == code  # still there
    ops.clear_device_error()
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("new,lens", [([1, 1, 1], [50, 20, 90]), ([40, 30, 1], [50, 70, 90])])
@pytest.mark.parametrize("where", ["own", "prefix"])
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
def test_a_bad_page_touches_its_request_alone(new, lens, where, bad):
    """Keys and values on a page outside the cache count as zeros; the other requests' rows are the same bits."""
    from distrain_b200 import ops
    from test_paged_gpu import Batch
    ops.clear_device_error()
    b = Batch(new, lens, 4, 2, 64, 16, pre=[40, 70], sizes=[1, 2], seed=2)
    clean = b.run()
    if where == "own":
        b.tables[0, 1] = bad
        b.ks[0][:, 16:32] = 0
        b.vs[0][:, 16:32] = 0
    else:
        b.prefix[0][0, 1] = bad
        b.pks[0][:, 16:32] = 0
        b.pvs[0][:, 16:32] = 0
    out = b.run()
    assert ops.device_error()[0] == 5
    ops.clear_device_error()
    assert torch.equal(out[new[0]:], clean[new[0]:])
    ref, size, _ = b.ref()
    # (the bound of an attention output: test_paged_gpu.py)
    assert ((out.double().view(ref.shape) - ref).abs() <= ref.abs() * 2 ** -8 + (2 ** -7 + 2 ** -13) * size + 1e-30).all()


# ───────────────────────── generation ─────────────────────────
def test_generation_fails_on_what_the_gpu_reports():
    """A page lost from a decoder's tables, a step its page tables refuse, and a request after each that is as before."""
    from distrain_b200 import ops
    from distrain_b200.serve import sample_cached
    from test_decode_gpu import _decoder
    ops.clear_device_error()
    _, _, dec = _decoder()
    ids = [3, 5, 7, 11, 13] * 9
    want = sample_cached(dec, ids, 2, 20)
    branch = dec.branch

    def lost(n):
        branch(n)
        dec.prefix[0, 1] = 10 ** 6

    def full(n):
        branch(n)
        dec.cached += 16 * dec.answer_pages  # a table row has no room behind these

    for bad, what, tokens in ((lost, "error 5", 20), (full, "page tables", 2)):
        dec.branch = bad
        with pytest.raises(RuntimeError, match=what):
            sample_cached(dec, ids, 2, tokens)
        dec.branch = branch
        assert ops.device_error() == (0, 0)
        assert sample_cached(dec, ids, 2, 20) == want


# ───────────────────────── buffers that share memory ─────────────────────────
def _zeros(*s, dtype=torch.bfloat16):
    return torch.zeros(*s, dtype=dtype, device=DEV)


def test_shifted_views_of_one_buffer_are_refused():
    """An output that begins at another element than an input, but lies over it."""
    from distrain_b200.ops import paged, sampling
    i32, f32 = torch.int32, torch.float32
    refused = lambda: pytest.raises(ValueError, match="share memory")  # noqa: E731
    # page tables: every output against an input and another output
    names = ["tables", "slots", "positions", "cu", "total", "used"]
    def tables(**kw):
        a = dict(cached=_zeros(8, dtype=i32), new=_zeros(8, dtype=i32), free=_zeros(9, dtype=i32), tables=_zeros(8, 4, dtype=i32),
                 slots=_zeros(8, dtype=i32), positions=_zeros(8, dtype=i32), cu=_zeros(9, dtype=i32),
                 total=_zeros(8, dtype=i32), used=_zeros(2, dtype=i32), start=_zeros(8, dtype=i32))
        for name, t in kw.items():
            assert t.shape == a[name].shape
        a.update(kw)
        paged.page_tables(**a, page_size=16)
    tables()
    sizes = dict(tables=32, slots=8, positions=8, cu=9, total=8, used=2, cached=8, new=8, free=9, start=8)
    for out in names:
        for other in ["cached", "new", "free", "start"] + [n for n in names if n != out]:
            buf = _zeros(64, dtype=i32)
            x, y = buf[:sizes[out]], buf[1:1 + sizes[other]]
            shape = lambda n, t: t.view(8, 4) if n == "tables" else t  # noqa: E731
            with refused():
                tables(**{out: shape(out, x), other: shape(other, y)})
    wide = _zeros(8, 16, dtype=i32)
    tables(tables=wide[:, :4], cu=wide[0, 4:13], total=wide[1, 4:12])  # in the gaps of the rows: not shared
    with refused():
        tables(tables=wide[:, :4], total=wide.view(-1)[28:36])  # into row 2
    # append
    d, P, nh, nkv, T = 32, 16, 4, 2, 4
    def append(**kw):
        a = dict(qkv=_zeros(T, 8 * d), bias=_zeros(8 * d, dtype=f32), cos=_zeros(8, 16, dtype=f32), sin=_zeros(8, 16, dtype=f32),
                 slots=_i([0, 1, 2, 3]), positions=_i([0, 1, 2, 3]), q=_zeros(T, nh * d), k_cache=_zeros(2, nkv, P, d),
                 v_cache=_zeros(2, nkv, P, d))
        a.update(kw)
        paged.kv_append(**a)
    append()
    k = _zeros(3, nkv, P, d)
    buf = _zeros(T * 8 * d + 8)
    for kw in (dict(k_cache=k[:2], v_cache=k[1:]), dict(k_cache=k[:2], v_cache=k[:2]),
               dict(qkv=buf[:T * 8 * d].view(T, 8 * d), q=buf[8:8 + T * nh * d].view(T, nh * d)),
               dict(qkv=k.view(-1)[8:8 + T * 8 * d].view(T, 8 * d), k_cache=k[:2])):
        with refused():
            append(**kw)
    # attention
    cu, lens, tb = _i([0, 4]), _i([4]), _i([[0]])
    def attend(groups=0, **kw):
        plan = paged.AttentionPlan(T, 1, groups, nh=nh, nkv=nkv, d=d, page_size=P)
        plan.build(cu, lens, tb, prefix=(_i([[1]]), _i([3]), _i([0, 1])) if groups else None)
        a = dict(q=_zeros(T, nh * d), k_cache=_zeros(2, nkv, P, d), v_cache=_zeros(2, nkv, P, d), out=_zeros(T, nh * d))
        a.update(kw)
        paged.paged_attention(plan=plan, **a)
    attend()
    attend(groups=1)
    both = _zeros(T * nh * d + 8)
    n = T * nh * d
    with refused():
        attend(q=both[:n].view(T, -1), out=both[8:8 + n].view(T, -1))
    with refused():
        attend(k_cache=k[:2], out=k.view(-1)[8:8 + n].view(T, -1))
    with refused():
        attend(q=both[:n].view(T, -1), lse=both.view(f32)[4:4 + T * nh].view(T, nh))
    with refused():
        attend(out=both[:n].view(T, -1), lse=both.view(f32)[4:4 + T * nh].view(T, nh))
    same = _zeros(2, nkv, P, d)
    attend(k_cache=same, v_cache=same)  # inputs may be one another
    # logits
    B, V = 4, 50
    z = _zeros(B * V + 4, dtype=f32)
    x, o = z[:B * V].view(B, V), z[4:4 + B * V].view(B, V)
    with refused():
        sampling.process_logits(x, o)
    sampling.process_logits(x, x)  # in place
    pair = _zeros(B, 2 * V, dtype=f32)
    pair.normal_()
    left = pair[:, :V].clone()
    sampling.process_logits(pair[:, :V], pair[:, V:])  # side by side
    assert torch.equal(pair[:, V:], left) and torch.equal(pair[:, :V], left)
    with refused():
        sampling.process_logits(pair[:, :V], pair[:, V - 1:2 * V - 1])
    with refused():
        sampling.process_logits(_zeros(B, V, dtype=f32), x, history=z.view(i32)[:B * 5].view(B, 5), lens=_i([1] * B))
    with refused():
        sampling.process_logits(_zeros(B, V, dtype=f32), x, mask=z.view(i32)[2:2 + B * 2].view(B, 2))
    with refused():
        sampling.process_logits(_zeros(B, V), x, history=_zeros(B, 5, dtype=i32), lens=_i([1] * B), presence=z[8:8 + B])


def test_rows_off_a_16_byte_boundary_are_refused():
    """Like every other argument that does not fit: a ValueError, and nothing written."""
    from distrain_b200.ops import paged
    d, P, nh, nkv, T = 32, 16, 4, 2, 4
    def view(*shape, dtype=torch.bfloat16, off=4):
        n = 1
        for s in shape:
            n *= s
        return torch.ones(n + 16, dtype=dtype, device=DEV)[off:off + n].view(*shape)
    off = dict(qkv=view(T, 8 * d), bias=view(8 * d, dtype=torch.float32, off=1), cos=view(8, 16, dtype=torch.float32, off=2),
               sin=view(8, 16, dtype=torch.float32, off=3), q=view(T, nh * d), k_cache=view(2, nkv, P, d),
               v_cache=view(2, nkv, P, d))
    for name, t in off.items():
        a = dict(qkv=_zeros(T, 8 * d), bias=None, cos=_zeros(8, 16, dtype=torch.float32),
                 sin=_zeros(8, 16, dtype=torch.float32), slots=_i([0, 1, 2, 3]), positions=_i([0, 1, 2, 3]), q=_zeros(T, nh * d),
                 k_cache=_zeros(2, nkv, P, d), v_cache=_zeros(2, nkv, P, d))
        a[name] = t
        with pytest.raises(ValueError, match="16-byte"):
            paged.kv_append(**a)
        assert (t == 1).all()
    plan = paged.AttentionPlan(T, 1, nh=nh, nkv=nkv, d=d, page_size=P)
    plan.build(_i([0, 4]), _i([4]), _i([[0]]))
    for name in ("q", "k_cache", "v_cache", "out"):
        a = dict(q=_zeros(T, nh * d), k_cache=_zeros(2, nkv, P, d), v_cache=_zeros(2, nkv, P, d), out=_zeros(T, nh * d))
        a[name] = view(*a[name].shape)
        with pytest.raises(ValueError, match="16-byte"):
            paged.paged_attention(plan=plan, **a)
        assert (a[name] == 1).all()


@pytest.mark.parametrize("scale", [1e-30, 1e-3])
def test_small_scales(scale):
    """Weights that are all alike, in both kernels, with rows that see nothing."""
    from test_paged_gpu import Batch
    Batch([1, 60, 3], [400, 90, 2], 4, 2, 64, 16).check(scale=scale)
    Batch([1, 60, 3], [400, 90, 2], 4, 2, 64, 16, pre=[70, 0], sizes=[2, 1]).check(scale=scale)


@pytest.mark.parametrize("cached,new", [(2 ** 31 - 10, 5), (2 ** 31 - 1, 0), (2 ** 31 - 17, 2), (0, 2 ** 31 - 1)])
def test_lengths_near_2_to_31_are_refused(cached, new):
    """A table row wide enough for them would otherwise be read and written at offsets that have wrapped."""
    from distrain_b200.ops import paged
    B, P, width = 2, 16, 2 ** 27 + 8
    tables = torch.full((B, width), 7, dtype=torch.int32, device=DEV)
    slots, pos = _i([99] * 8), _i([99] * 8)
    cu, total, used = _i([99] * 3), _i([99] * 2), _i([99, 99])
    paged.page_tables(_i([3, cached]), _i([1, new]), torch.arange(9, dtype=torch.int32, device=DEV), tables, slots, pos, cu,
                      total, used, page_size=P)
    assert used[0] == 0 and used.tolist()[1] & paged.TABLE_FULL
    assert cu.tolist() == [0, 0, 0] and total.tolist() == [3, cached] and slots.tolist() == [-1] * 8
    assert bool((tables == 7).all())


@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (4, 2, 32), (16, 4, 128)])
@pytest.mark.parametrize("new,lens,pre,sizes", [([1, 1], [51, 70], [], []), ([30, 2], [80, 52], [], []),
                                                ([1, 2, 1], [51, 60, 9], [40, 30], [2, 1]),
                                                ([20, 9, 1], [70, 59, 51], [300, 90], [2, 1])])
@pytest.mark.parametrize("where", ["own", "last", "prefix"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_key_that_is_no_number_reaches_what_sees_it(nh, nkv, d, new, lens, pre, sizes, where, value):
    """One element of one key of kv head 1: the query heads on it become NaN for the tokens that see the key, and every
    other row is the same bits as without it."""
    from test_paged_gpu import Batch
    if where == "prefix" and not pre:
        return
    b = Batch(new, lens, nh, nkv, d, 16, pre=pre, sizes=sizes, seed=3)
    b.q.abs_()  # (an infinite product has one sign: scores of +inf, whose softmax is NaN)
    clean = b.run()
    if where == "prefix":
        b.k[int(b.prefix[0][0, 1]), 1, 3, 5] = value
        hit = list(range(sum(new[:sizes[0]])))
    else:
        at = lens[0] - 1 if where == "last" else 20  # its last key is seen by the last token alone
        b.k[int(b.tables[0, at // 16]), 1, at % 16, 5] = value
        hit = [j for j in range(new[0]) if lens[0] - new[0] + j >= at]
    out = b.run()
    assert hit and len(hit) < sum(new)
    o, c = out.view(-1, nkv, nh // nkv * d), clean.view(-1, nkv, nh // nkv * d)
    assert torch.isnan(o[hit, 1]).all()
    o[hit, 1] = c[hit, 1]
    assert torch.equal(o, c)


def test_requests_at_once_and_from_the_command_line(tmp_path, capsys):
    """HTTP requests that arrive together, on handler threads, give what they give one by one; generate takes a device
    without an index and refuses a token that the vocabulary does not have."""
    import concurrent.futures
    import json
    import urllib.error
    import urllib.request
    from distrain_b200.cli import main
    from distrain_b200.serve import CompletionServer
    from distrain_b200.utils.checkpoint import save_safetensors
    from test_decode_gpu import _decoder
    _, sd, _ = _decoder(vocab=512)
    path = str(tmp_path / "m.safetensors")
    save_safetensors(sd, path)
    srv = CompletionServer(path, device="cuda", max_tokens_cap=32, kv_cache=True, max_n=4)
    port = srv.start("127.0.0.1", 0, threads=4)

    def post(body):
        req = urllib.request.Request(f"http://127.0.0.1:{port}/v1/completions", method="POST", data=json.dumps(body).encode())
        try:
            with urllib.request.urlopen(req, timeout=60) as r:
                return r.status, json.loads(r.read())["choices"]
        except urllib.error.HTTPError as e:
            return e.code, None
    bodies = [{"prompt": [1 + i, 2, 3] * (1 + 20 * i), "max_tokens": 20, "n": 1 + i % 3, "temperature": 0.7 * (i % 2), "seed": i,
               "presence_penalty": 0.5 * (i // 3)} for i in range(6)]
    bodies += [{"prompt": [512], "max_tokens": 2}, {"prompt": [1], "max_tokens": 2, "presence_penalty": 1e39}]
    try:
        one_by_one = [post(b) for b in bodies]
        assert [s for s, _ in one_by_one] == [200] * 6 + [400] * 2
        with concurrent.futures.ThreadPoolExecutor(8) as pool:
            assert list(pool.map(post, bodies)) == one_by_one
    finally:
        srv.stop()
    main(["generate", path, "--prompt-ids", "5,6,7", "--max-tokens", "4", "--device", "cuda", "--kv-cache"])
    ids = json.loads(capsys.readouterr().out.strip().splitlines()[-1])["ids"]
    assert ids[:3] == [5, 6, 7] and len(ids) == 7
    with pytest.raises(ValueError, match="vocabulary"):
        main(["generate", path, "--prompt-ids", "5,512", "--max-tokens", "4", "--device", "cuda", "--kv-cache"])
