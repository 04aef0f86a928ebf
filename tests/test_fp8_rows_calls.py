"""Calls of the 8-bit row functions (vectors_b200/fp8.py, include/vx.h) that their documentation allows and
that are easily got wrong: calls with nothing to do, all operand types in every form, repeated and
concurrent small calls.  The definition and the tolerances are those of test_fp8_rows.py.
"""
import numpy as np
import pytest

import vectors_b200 as vx
import vectors_b200._native as N
from tests.test_fp8_rows import _bytes, _dtype, _grouped_want, _store, bound, decode, encode, rows_of


STAR = """
import sys
if {blocked}:
    sys.modules["torch"] = None  # as where it is not installed: importing it raises ImportError
from vectors_b200 import *
import vectors_b200
assert {blocked} or "torch" not in sys.modules
assert all(n in globals() for n in vectors_b200.__all__) and "FlatScanAdapter" in globals()
try:
    assert fp8_pitch(513) == (640, 8) == vectors_b200.fp8_pitch(513)
    assert not {blocked} and "torch" in sys.modules
    assert vectors_b200.fp8_pitch is vectors_b200.fp8.fp8_pitch
    try:
        fp8_empty(capacity=-1, dim=100, device="cpu")
    except IllegalArgumentException:
        print("star: ok")
except ImportError:
    assert {blocked}
    print("star: ok")
"""


@pytest.mark.parametrize("blocked", [False, True])
def test_star_import_without_torch(blocked):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", STAR.format(blocked=blocked)], cwd=root, capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0 and "star: ok" in run.stdout, run.stdout + run.stderr


class _OnDevice:
    """A host tensor that says it is on device 0: what these calls refuse, they refuse before any use of it."""

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return 0

    def is_contiguous(self):
        return self.t.is_contiguous()

    def contiguous(self):
        return self


def _refused(monkeypatch, call):
    """The message of a call that is refused before it reaches the library."""
    import vectors_b200.fp8 as fp8

    monkeypatch.setattr(fp8, "_call", lambda name: pytest.fail(f"{name} was called"))
    monkeypatch.setattr(fp8, "_raw_stream", lambda device: 0)
    with pytest.raises(vx.IllegalArgumentException) as e:
        call()
    return str(e.value)


def _host_store(capacity, dim):
    codes, scales = vx.fp8_empty(capacity, dim, device="cpu")
    return _OnDevice(codes), _OnDevice(scales)


@pytest.mark.parametrize("first", [-1, 8, 1 << 31, 1 << 63, 1 << 64, -(1 << 64), (1 << 64) + 2])
def test_first_row_out_of_the_store(monkeypatch, first):
    """Also numbers that 64 bits would wrap into the store."""
    import torch

    codes, scales = _host_store(10, 100)
    rows = _OnDevice(torch.zeros(3, 100))
    assert "store of 10" in _refused(monkeypatch, lambda: vx.fp8_write_device(rows, codes, scales, first=first))
    out = _OnDevice(torch.zeros(3, 100))
    assert "store of 10" in _refused(monkeypatch, lambda: vx.fp8_read_device(codes, scales, 100, first=first, count=3, out=out))


def test_first_row_with_slots(monkeypatch):
    import torch

    codes, scales = _host_store(10, 100)
    rows, slots = _OnDevice(torch.zeros(3, 100)), _OnDevice(torch.zeros(3, dtype=torch.int64))
    message = _refused(monkeypatch, lambda: vx.fp8_write_device(rows, codes, scales, slots=slots, first=2))
    assert "exclude" in message
    message = _refused(monkeypatch, lambda: vx.fp8_read_device(codes, scales, 100, slots=slots, first=2, out=rows))
    assert "exclude" in message


def test_check_of_a_device_that_is_not_there():
    """The framework's own exceptions, not torch's."""
    if vx.device_count() == 0:
        with pytest.raises(vx.GpuUnavailableException):
            vx.fp8_check()
    for device in (-1, 63, 64):
        with pytest.raises((vx.IllegalArgumentException, vx.GpuUnavailableException)):
            vx.fp8_check(device)


@pytest.mark.gpu
@pytest.mark.parametrize("max_rows", [5, 0])
def test_no_groups_and_no_offsets(max_rows):
    """No groups need no offsets, and leave the results as they are (which have a column for every stored
    row here, more than max_rows)."""
    import torch

    codes, scales = vx.fp8_empty(40, 100)
    q = torch.randn(3, 100, device="cuda")
    out = torch.full((3, 40), -7.0, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for offsets in (None, torch.zeros(1, dtype=torch.int64, device="cuda").data_ptr()):
        status = N.lib().vx_fp8_scores_grouped_device(0, q.data_ptr(), N.VX_F32, None, 3, 100, offsets, codes.data_ptr(),
                                                      scales.data_ptr(), 40, offsets, 0, 100, out.data_ptr(), N.VX_F32, 40,
                                                      max_rows, stream)
        assert status == 0, N.last_error()
    vx.fp8_check()
    assert (out == -7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [1, 8, 74, 75, 200])
def test_small_grouped_calls_one_after_another(groups):
    """Fewer tiles than clusters (74 on a B200), as many, and a few more: hundreds of calls queued on three
    streams, so that clusters of one call start where those of another have just ended."""
    import torch

    dim, per = 128, 7
    q, x = rows_of(groups, dim, groups, 1.0), rows_of(groups * per, dim, groups + 1, 1.0)
    codes, scales = _store(x)
    qo, ro = np.arange(groups + 1), np.arange(groups + 1) * per
    want, tol = _grouped_want(decode(*encode(q)), decode(_bytes(codes), scales.cpu().numpy()), qo, ro, per, 0.0)
    tq, tqo, tro = torch.from_numpy(q).cuda(), torch.from_numpy(qo).cuda(), torch.from_numpy(ro).cuda()
    qc, qs = _store(q)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for i in range(300):
        with torch.cuda.stream(streams[i % 3]):
            if i % 2:
                outs.append(vx.fp8_scores_grouped_device(qc, tqo, codes, scales, tro, query_scales=qs, max_rows=per))
            else:
                outs.append(vx.fp8_scores_grouped_device(tq, tqo, codes, scales, tro, max_rows=per))
    torch.cuda.synchronize()
    vx.fp8_check()
    assert (np.abs(outs[0].cpu().numpy() - want) <= tol).all()
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [128, 512, 640, 1500, 1664, 4000])
def test_short_calls_of_every_pipeline_depth(dim):
    """Products of fewer chunks than the pipeline has stages, as many and more, queued on three streams so that
    clusters of one call start where those of another have just ended."""
    import torch

    q, x = rows_of(50, dim, 3, 1.0), rows_of(700, dim, 4, 1.0)
    codes, scales = _store(x)
    qc, qs = _store(q)
    dq, dr = decode(*encode(q)), decode(_bytes(codes), scales.cpu().numpy())
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i in range(150):
        with torch.cuda.stream(streams[i % 3]):
            got.append(vx.fp8_scores_device(qc, codes, scales, query_scales=qs))
    torch.cuda.synchronize()
    vx.fp8_check()
    assert (np.abs(got[0].cpu().numpy() - dq @ dr.T) <= bound(dq, dr, "float32")).all()
    assert all(torch.equal(g, got[0]) for g in got)


@pytest.mark.gpu
@pytest.mark.parametrize("nq, dim", [(1, 768), (20, 500), (64, 256)])
def test_few_queries_that_change_from_call_to_call(nq, dim):
    """Few float queries are quantised inside the product, by both CTAs of each cluster for its tensor cores:
    calls in a row on other queries each see their own (a stale code or scale is another call's)."""
    import torch

    x = rows_of(30000, dim, 1)
    codes, scales = _store(x)
    sets = [torch.from_numpy(rows_of(nq, dim, 10 + s)).cuda() for s in range(4)]
    want = []
    for q in sets:
        qc, qs = vx.fp8_empty(nq, dim)
        vx.fp8_write_device(q, qc, qs)
        want.append(vx.fp8_scores_device(qc, codes, scales, query_scales=qs))
    for n in (30000, 1000):
        got = [vx.fp8_scores_device(sets[i % 4], codes[:n], scales[:n]) for i in range(100)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, want[i % 4][:, :n]) for i, g in enumerate(got))
    vx.fp8_check()


@pytest.mark.gpu
@pytest.mark.parametrize("nq, n, dim", [(3, 9000, 2048), (200, 3000, 4096), (130, 5000, 600)])
def test_scales_that_change_from_slot_to_slot(nq, n, dim):
    """Scales far apart from block to block and from call to call, copied by both CTAs of each cluster for its
    tensor cores: a scale of an earlier slot or call would be off by powers of two."""
    import torch

    stores = [_store(rows_of(n, dim, 30 + s, 6.0)) for s in range(2)]
    queries = [_store(rows_of(nq, dim, 40 + s, 6.0)) for s in range(2)]
    got = [vx.fp8_scores_device(queries[i % 2][0], *stores[i // 2 % 2], query_scales=queries[i % 2][1]) for i in range(60)]
    torch.cuda.synchronize()
    vx.fp8_check()
    for i in range(4):
        dq = decode(_bytes(queries[i % 2][0]), queries[i % 2][1].cpu().numpy())
        dr = decode(_bytes(stores[i // 2][0]), stores[i // 2][1].cpu().numpy())
        assert (np.abs(got[i].cpu().numpy() - dq @ dr.T) <= bound(dq, dr, "float32")).all()
        assert all(torch.equal(g, got[i]) for g in got[i::4])


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("queries", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("view", ["whole", "half_aligned", "shifted"])
@pytest.mark.parametrize("groups, nq, n, dim", [(6, 700, 1500, 256), (40, 90, 3000, 200), (3, 5, 1100, 640), (300, 2000, 1200, 96)])
def test_grouped_values_of_every_type(groups, nq, n, dim, view, queries, out):
    """Queries of each type, with rows that every load width starts at, and results of each type: the values of
    every group, what lies past a group's rows kept in a given result and zero in a new one."""
    import torch

    r = np.random.default_rng(groups)
    q, x = rows_of(nq, dim + 4, groups, 1.0), rows_of(n, dim, groups + 1, 1.0)
    # elements from one query to the next and the first one's place: 16-byte loads, 8-byte loads, single elements
    wide = torch.from_numpy(q).cuda().to(_dtype(queries))
    tq = {"whole": wide[:, :dim].contiguous(), "half_aligned": wide[:, 4:], "shifted": wide[:, 1 : dim + 1]}[view]
    qo = np.sort(np.concatenate([[0, nq], r.integers(0, nq + 1, groups - 1)]))
    ro = np.sort(np.concatenate([[0, n], r.integers(0, n + 1, groups - 1)]))
    codes, scales = _store(x)
    dq, dr = decode(*encode(tq.float().cpu().numpy())), decode(_bytes(codes), scales.cpu().numpy())
    width = int((ro[1:] - ro[:-1]).max())
    tqo, tro = torch.from_numpy(qo).cuda(), torch.from_numpy(ro).cuda()
    value = np.zeros((nq, width))
    tol, inside = np.zeros((nq, width)), np.zeros((nq, width), bool)
    for g in range(groups):
        a, b, c, d = qo[g], qo[g + 1], ro[g], ro[g + 1]
        if a < b and c < d:
            value[a:b, : d - c] = dq[a:b] @ dr[c:d].T
            tol[a:b, : d - c] = bound(dq[a:b], dr[c:d], out)
            inside[a:b, : d - c] = True
    given = torch.full((nq, width), -3.0, dtype=_dtype(out), device="cuda")
    fresh = vx.fp8_scores_grouped_device(tq, tqo, codes, scales, tro, max_rows=width, dtype=_dtype(out))
    assert vx.fp8_scores_grouped_device(tq, tqo, codes, scales, tro, out=given) is given
    for got, past in ((given, -3.0), (fresh, 0.0)):
        assert got.dtype == _dtype(out)
        err = np.abs(got.float().cpu().numpy().astype(np.float64) - np.where(inside, value, past))
        assert (err <= tol).all(), (err.max(), np.argwhere(err > tol)[:5])


@pytest.mark.gpu
@pytest.mark.parametrize("call", ["write", "read", "few", "many", "stored", "grouped", "check"])
def test_first_cuda_call_of_a_thread(call):
    """Each function as the first CUDA call that a thread makes (it has no current context yet)."""
    import threading

    import torch

    x, q = torch.from_numpy(rows_of(500, 100, 1)).cuda(), torch.from_numpy(rows_of(300, 100, 2)).cuda()
    codes, scales = vx.fp8_empty(500, 100)
    vx.fp8_write_device(x, codes, scales)
    c2, s2 = vx.fp8_empty(500, 100)
    off = torch.tensor([0, 300], device="cuda"), torch.tensor([0, 500], device="cuda")
    back, out = torch.empty_like(x), torch.empty(300, 500, device="cuda")
    calls = {"write": lambda: vx.fp8_write_device(x, c2, s2), "read": lambda: vx.fp8_read_device(codes, scales, 100, out=back),
             "few": lambda: vx.fp8_scores_device(q[:3], codes, scales, out=out[:3]),
             "many": lambda: vx.fp8_scores_device(q, codes, scales, out=out),
             "stored": lambda: vx.fp8_scores_device(codes[:300], codes, scales, query_scales=scales[:300], out=out),
             "grouped": lambda: vx.fp8_scores_grouped_device(q, off[0], codes, scales, off[1], out=out),
             "check": lambda: vx.fp8_check()}
    torch.cuda.synchronize()
    failed = []

    def work():
        try:
            calls[call]()
        except Exception as e:
            failed.append(e)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not failed
    if call == "write":
        assert torch.equal(c2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s2, scales)
    elif call == "read":
        assert torch.equal(back, vx.fp8_read_device(codes, scales, 100))
    elif call in ("few", "many", "grouped"):
        n = 3 if call == "few" else 300
        assert torch.equal(out[:n], vx.fp8_scores_device(q[:n], codes, scales))
    elif call == "stored":
        assert torch.equal(out, vx.fp8_scores_device(codes[:300], codes, scales, query_scales=scales[:300]))


def test_wait_limit_of_the_hook_is_validated():
    for limit_ms in (0, 20000):
        assert N.lib().vx_debug_fp8_wait_timeout(0, limit_ms, None) == N.VX_ERR_INVALID_ARGUMENT
    assert N.lib().vx_debug_fp8_wait_timeout(-1, 20, None) == N.VX_ERR_INVALID_ARGUMENT


@pytest.mark.gpu
def test_a_wait_that_ran_out_is_reported_once():
    """By fp8_check, or by the next product, which leaves its results as they are; the one after works."""
    import torch

    q, x = rows_of(3, 100, 1), rows_of(50, 100, 2)
    codes, scales = _store(x)
    tq = torch.from_numpy(q).cuda()
    want = vx.fp8_scores_device(tq, codes, scales)
    offsets = torch.tensor([0, 3], device="cuda"), torch.tensor([0, 50], device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    vx.fp8_check()
    assert N.lib().vx_debug_fp8_wait_timeout(0, 20, stream) == 0, N.last_error()
    with pytest.raises(vx.GpuUnavailableException, match="time budget"):
        vx.fp8_check()
    vx.fp8_check()
    for call in (lambda o: vx.fp8_scores_device(tq, codes, scales, out=o),
                 lambda o: vx.fp8_scores_grouped_device(tq, offsets[0], codes, scales, offsets[1], out=o)):
        out = torch.full((3, 50), -7.0, device="cuda")
        assert N.lib().vx_debug_fp8_wait_timeout(0, 20, stream) == 0
        torch.cuda.synchronize()
        with pytest.raises(vx.GpuUnavailableException, match="time budget"):
            call(out)
        assert (out == -7).all()
        assert torch.equal(call(out), want)
    vx.fp8_check()


@pytest.mark.gpu
def test_a_wait_that_ran_out_is_reported_to_one_of_many_threads():
    import threading

    import torch

    codes, scales = _store(rows_of(50, 100, 2))
    q = torch.from_numpy(rows_of(3, 100, 1)).cuda()
    want = vx.fp8_scores_device(q, codes, scales)
    for _ in range(20):
        assert N.lib().vx_debug_fp8_wait_timeout(0, 1, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        start, reports, results = threading.Barrier(8), [], []

        def work():
            start.wait()
            try:
                results.append(vx.fp8_scores_device(q, codes, scales))
            except vx.GpuUnavailableException as e:
                reports.append(str(e))

        threads = [threading.Thread(target=work) for _ in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert len(reports) == 1 and "time budget" in reports[0]
        assert len(results) == 7 and all(torch.equal(r, want) for r in results)


@pytest.mark.gpu
def test_negated_views():
    """torch keeps the imaginary part of a conjugate as a view with a flag and the other sign's bits."""
    import torch

    z = torch.complex(torch.zeros(40, 1), torch.from_numpy(rows_of(40, 1, 1))).cuda()
    x = z.conj().imag
    assert x.is_neg()
    codes, scales = vx.fp8_empty(40, 1)
    vx.fp8_write_device(x, codes, scales)
    c, s = encode(x.cpu().numpy())
    assert np.array_equal(_bytes(codes), c) and np.array_equal(scales.cpu().numpy(), s)
    d = decode(c, s)
    got = vx.fp8_scores_device(x, codes, scales)
    assert (np.abs(got.cpu().numpy() - d @ d.T) <= bound(d, d, "float32")).all()
    with pytest.raises(vx.IllegalArgumentException, match="negated"):
        vx.fp8_read_device(codes, scales, 1, out=x)


@pytest.mark.gpu
def test_one_row_broadcast_in_one_dimension():
    import torch

    x = torch.full((1, 1), 3.25, device="cuda").expand(9, 1)
    codes, scales = vx.fp8_empty(9, 1)
    vx.fp8_write_device(x, codes, scales)
    assert (vx.fp8_read_device(codes, scales, 1) == 3.25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [65536, 65409])
def test_largest_dimension(dim):
    """Rows of 512 blocks: written, read back, and scored for float and stored queries, alone and in groups."""
    import torch

    q, x = rows_of(5, dim, 1, 1.0), rows_of(300, dim, 2, 1.0)
    tq = torch.from_numpy(q).cuda()
    codes, scales = vx.fp8_empty(300, dim)
    vx.fp8_write_device(torch.from_numpy(x).cuda(), codes, scales, slots=torch.arange(299, -1, -1, device="cuda"))
    c, s = encode(x[::-1])
    assert np.array_equal(_bytes(codes), c) and np.array_equal(scales.cpu().numpy(), s)
    dr, dq = decode(c, s), decode(*encode(q))
    assert np.array_equal(vx.fp8_read_device(codes, scales, dim, first=297).cpu().numpy(), dr[297:, :dim].astype(np.float32))
    want, tol = dq @ dr.T, bound(dq, dr, "float32")
    got = vx.fp8_scores_device(tq, codes, scales)
    assert (np.abs(got.cpu().numpy() - want) <= tol).all()
    qc, qs = _store(q)
    assert torch.equal(vx.fp8_scores_device(qc, codes, scales, query_scales=qs), got)
    assert torch.equal(vx.fp8_scores_device(tq[:1], codes, scales), got[:1])
    grouped = vx.fp8_scores_grouped_device(tq, torch.tensor([0, 2, 5], device="cuda"), codes, scales,
                                           torch.tensor([0, 17, 300], device="cuda"), max_rows=283)
    assert torch.equal(grouped[:2, :17], got[:2, :17]) and torch.equal(grouped[2:], got[2:, 17:])


@pytest.mark.gpu
def test_writes_and_products_of_many_threads():
    """Four threads, each on its stream, mixing writes to slots, reads and all forms of products: clusters of one
    call start on processors that another's are just leaving.  Every result has the bits of the same call alone."""
    import threading

    import torch

    r = np.random.default_rng(3)
    n, dim = 3000, 300
    x, q = torch.from_numpy(rows_of(n, dim, 1)).cuda(), torch.from_numpy(rows_of(200, dim, 2)).cuda()
    codes, scales = vx.fp8_empty(n, dim)
    vx.fp8_write_device(x, codes, scales)
    slots = torch.from_numpy(r.permutation(n + 500)[:n]).cuda()
    qo = torch.from_numpy(np.sort(np.concatenate([[0, 200], r.integers(0, 201, 29)]))).cuda()
    ro = torch.from_numpy(np.sort(np.concatenate([[0, n], r.integers(0, n + 1, 29)]))).cuda()

    def write():
        c, s = vx.fp8_empty(n + 500, dim)
        vx.fp8_write_device(x, c, s, slots=slots)
        return c.view(torch.uint8), s

    calls = [write, lambda: (vx.fp8_read_device(codes, scales, dim, slots=slots),),
             lambda: (vx.fp8_scores_device(q[:2], codes, scales),), lambda: (vx.fp8_scores_device(q, codes, scales),),
             lambda: (vx.fp8_scores_device(codes[:50], codes, scales, query_scales=scales[:50]),),
             lambda: (vx.fp8_scores_grouped_device(q, qo, codes, scales, ro, max_rows=n),)]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    failed = []

    def work(seed):
        pick = np.random.default_rng(seed)
        stream = torch.cuda.Stream()
        try:
            with torch.cuda.stream(stream):
                for _ in range(100):
                    ids = pick.integers(0, len(calls), 20)
                    got = [calls[i]() for i in ids]
                    stream.synchronize()
                    for i, g in zip(ids, got):
                        if not all(torch.equal(a, b) for a, b in zip(g, want[i])):
                            failed.append(int(i))
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(seed,)) for seed in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    vx.fp8_check()
    assert not failed
