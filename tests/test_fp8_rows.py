"""Rows in 8 bits (vectors_b200/fp8.py): quantising as rows are written, reading back, and the score
products, against the definition in 64 bits.

Tolerances.  Codes, scales and read-back values are exact.  A score is a sum of K exact products in
fp32: fewer than K additions, each off by at most one unit in the last place of a partial sum
(truncation included), so |error| <= K * 2^-23 * sum |q_k r_k|; an fp16 / bf16 result is rounded
once more, by 2^-11 / 2^-8 of the value.
"""
import numpy as np
import pytest

import vectors_b200 as vx

BLOCK = 128


# ---------------------------------------------------------------- the definition, in 64 bits
def e4m3_values():
    """Value of every e4m3 code (no infinities; 0x7f and 0xff are NaN)."""
    v = np.empty(256)
    for c in range(256):
        s, e, m = -1.0 if c & 0x80 else 1.0, (c >> 3) & 15, c & 7
        v[c] = s * ((m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    v[0x7F] = v[0xFF] = np.nan
    return v


VALUES = e4m3_values()


def encode(x):
    """(codes uint8, scales uint8) of rows: the nearest value, ties to the even code, found by bisection in
    the sorted list of values."""
    x = np.asarray(x, np.float64)
    n, dim = x.shape
    nb = -(-dim // BLOCK)
    p = np.zeros((n, nb * BLOCK))
    p[:, :dim] = x
    p = p.reshape(n, nb, BLOCK)
    with np.errstate(invalid="ignore"):
        bad = ~np.isfinite(p).all(2)
    top = np.abs(np.where(bad[:, :, None], 0.0, p)).max(2)
    e = np.full((n, nb), -127)
    for i, j in zip(*np.nonzero(top)):
        k = -127
        while 448.0 * 2.0 ** k < top[i, j]:
            k += 1
        e[i, j] = k
    y = np.where(bad[:, :, None], 0.0, p) / 2.0 ** e.astype(np.float64)[:, :, None]
    grid = VALUES[:127]  # 0 .. 448, ascending
    a = np.abs(y)
    hi = np.clip(np.searchsorted(grid, a, "left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    down, up = a - grid[lo], grid[hi] - a
    pick = np.where(down < up, lo, np.where(up < down, hi, np.where(lo % 2 == 0, lo, hi)))
    codes = (pick | np.where(np.signbit(y), 0x80, 0)).astype(np.uint8)
    codes[bad] = 0x7F
    scales = np.zeros((n, -(-nb // 4) * 4), np.uint8)
    scales[:, :nb] = np.where(bad, 255, e + 127)
    return codes.reshape(n, nb * BLOCK), scales


def decode(codes, scales):
    n, kp = codes.shape
    nb = kp // BLOCK
    s = np.where(scales[:, :nb] == 255, np.nan, 2.0 ** (scales[:, :nb].astype(np.float64) - 127))
    return (VALUES[codes].reshape(n, nb, BLOCK) * s[:, :, None]).reshape(n, kp)


def rows_of(n, dim, seed, spread=3.0):
    """Rows whose blocks differ in magnitude by factors of 2^spread and more."""
    r = np.random.default_rng(seed)
    nb = -(-dim // BLOCK)
    m = np.repeat(2.0 ** (spread * r.standard_normal((n, nb))), BLOCK, axis=1)[:, :dim]
    return (r.standard_normal((n, dim)) * m).astype(np.float32)


def bound(q, r, out):
    """Allowed error of each score, from the decoded operands and the output type."""
    value = np.abs(q @ r.T)
    acc = q.shape[1] * 2.0 ** -23 * (np.abs(q) @ np.abs(r).T)
    half = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[out]
    tiny = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}[out]
    return acc + half * (value + acc) + tiny


# ---------------------------------------------------------------- without a GPU
def test_definition_of_the_values():
    assert VALUES[0x7E] == 448 and VALUES[1] == 2.0 ** -9 and VALUES[0x38] == 1.0
    codes, scales = encode(np.array([[448.0, 449.0 / 1024]]))
    assert scales[0, 0] == 127 and codes[0, 0] == 0x7E
    codes, scales = encode(np.array([[448.5]]))
    assert scales[0, 0] == 128 and VALUES[codes[0, 0]] == 224.0


def test_pitch():
    assert vx.fp8_pitch(1) == (128, 4)
    assert vx.fp8_pitch(128) == (128, 4)
    assert vx.fp8_pitch(513) == (640, 8)
    assert vx.fp8_pitch(65536) == (65536, 512)
    for d in (0, -1, 65537):
        with pytest.raises(vx.IllegalArgumentException):
            vx.fp8_pitch(d)
    import ctypes as C

    import vectors_b200._native as N

    for d in (1, 127, 128, 129, 512, 513, 768, 65536):
        a, b = C.c_int32(), C.c_int32()
        assert N.lib().vx_fp8_pitch(d, C.byref(a), C.byref(b)) == 0
        assert (a.value, b.value) == vx.fp8_pitch(d)
    assert N.lib().vx_fp8_pitch(0, C.byref(a), C.byref(b)) == N.VX_ERR_INVALID_ARGUMENT
    assert N.lib().vx_fp8_pitch(8, None, C.byref(b)) == N.VX_ERR_NULL_POINTER


#: an address that passes the alignment checks and is never used: every call below is refused first
P = 1 << 20

WRITE = dict(device=0, rows=P, type=0, n=4, dim=100, row_stride=100, slots=None, slot_bytes=8, first=0, codes=P, scales=P,
             capacity=10, stream=None)
READ = dict(device=0, codes=P, scales=P, capacity=10, dim=100, slots=None, slot_bytes=8, first=0, n=4, out=P, out_type=0,
            out_stride=100, stream=None)
SCORES = dict(device=0, queries=P, query_type=0, query_scales=None, nq=3, query_stride=100, codes=P, scales=P, n=10, dim=100,
              out=P, out_type=0, out_stride=10, stream=None)
GROUPED = dict(device=0, queries=P, query_type=0, query_scales=None, nq=3, query_stride=100, query_offsets=P, codes=P,
               scales=P, n=10, row_offsets=P, groups=2, dim=100, out=P, out_type=0, out_stride=10, max_rows=10, stream=None)
BAD, NULL = 1, 2


@pytest.mark.parametrize("call, change, status", [
    ("write", dict(dim=0), BAD), ("write", dict(dim=65537, row_stride=1 << 20), BAD), ("write", dict(codes=None), NULL),
    ("write", dict(scales=None), NULL), ("write", dict(codes=P + 8), BAD), ("write", dict(scales=P + 2), BAD),
    ("write", dict(rows=None), NULL), ("write", dict(rows=P + 2), BAD), ("write", dict(type=1, rows=P + 1), BAD),
    ("write", dict(type=3), BAD), ("write", dict(type=-1), BAD), ("write", dict(row_stride=99), BAD),
    ("write", dict(n=-1), BAD), ("write", dict(first=-1), BAD), ("write", dict(first=7), BAD),
    ("write", dict(first=1 << 62), BAD), ("write", dict(capacity=-1), BAD), ("write", dict(capacity=1 << 31), BAD),
    ("write", dict(slots=P, slot_bytes=2), BAD), ("write", dict(slots=P + 4), BAD), ("write", dict(n=1 << 31, slots=P), BAD),
    ("write", dict(row_stride=1 << 62), BAD), ("write", dict(device=-1), BAD), ("write", dict(device=64), BAD),
    ("read", dict(out=None), NULL), ("read", dict(out_type=3), BAD), ("read", dict(out_stride=99), BAD),
    ("read", dict(n=11), BAD), ("read", dict(first=9, n=2), BAD), ("read", dict(codes=P + 1), BAD),
    ("read", dict(slots=P + 2, slot_bytes=4), BAD), ("read", dict(codes=None), NULL),
    ("scores", dict(nq=0), BAD), ("scores", dict(nq=-1), BAD), ("scores", dict(queries=None), NULL),
    ("scores", dict(query_stride=99), BAD), ("scores", dict(query_type=7), BAD), ("scores", dict(out=None), NULL),
    ("scores", dict(out_stride=9), BAD), ("scores", dict(out_type=3), BAD), ("scores", dict(out=P + 1), BAD),
    ("scores", dict(query_type=3), NULL), ("scores", dict(query_type=3, query_scales=P, queries=P + 8), BAD),
    ("scores", dict(codes=P + 8), BAD), ("scores", dict(scales=None), NULL), ("scores", dict(n=-1), BAD),
    ("grouped", dict(groups=-1), BAD), ("grouped", dict(query_offsets=None), NULL), ("grouped", dict(row_offsets=None), NULL),
    ("grouped", dict(row_offsets=P + 4), BAD), ("grouped", dict(max_rows=-1), BAD), ("grouped", dict(out_stride=9), BAD),
    ("grouped", dict(query_type=3, query_scales=P + 1), BAD),
])
def test_refusals_of_the_c_calls(call, change, status):
    import vectors_b200._native as N

    base, name = {"write": (WRITE, "vx_fp8_write_device"), "read": (READ, "vx_fp8_read_device"),
                  "scores": (SCORES, "vx_fp8_scores_device"), "grouped": (GROUPED, "vx_fp8_scores_grouped_device")}[call]
    got = getattr(N.lib(), name)(*{**base, **change}.values())
    assert got == status, N.last_error()
    assert N.last_error()


def test_injected_failure():
    import vectors_b200._native as N

    N.lib().vx_debug_fail_next(N.VX_ERR_OUT_OF_MEMORY)
    assert N.lib().vx_fp8_write_device(*WRITE.values()) == N.VX_ERR_OUT_OF_MEMORY


def test_refusals_of_host_tensors():
    import torch

    codes, scales = vx.fp8_empty(4, 100, device="cpu")
    assert codes.shape == (4, 128) and codes.dtype == torch.float8_e4m3fn and scales.shape == (4, 4)
    x = torch.zeros(4, 100)
    with pytest.raises(vx.IllegalArgumentException, match="CUDA"):
        vx.fp8_write_device(x, codes, scales)
    with pytest.raises(vx.NullPointerException):
        vx.fp8_scores_device(x, None, scales)
    with pytest.raises(vx.IllegalArgumentException, match="uint8"):
        vx.fp8_read_device(codes, scales.int(), 100)
    with pytest.raises(vx.IllegalArgumentException, match="float8"):
        vx.fp8_read_device(codes.float(), scales, 100)
    with pytest.raises(vx.IllegalArgumentException, match="must be \\[4\\]\\[4\\]"):
        vx.fp8_read_device(codes, scales[:, :3], 100)
    with pytest.raises(vx.IllegalArgumentException, match="multiple of 128"):
        vx.fp8_read_device(codes[:, :100], scales, 100)
    with pytest.raises(vx.IllegalArgumentException):
        vx.fp8_empty(-1, 100, device="cpu")


# ---------------------------------------------------------------- on the GPU: write and read
def _dtype(name):
    import torch

    return getattr(torch, name)


def _store(x, device="cuda"):
    """A store that holds the definition's codes of rows x."""
    import torch

    c, s = encode(x)
    return torch.from_numpy(c).to(device).view(torch.float8_e4m3fn), torch.from_numpy(s).to(device)


def _bytes(codes):
    import torch

    return codes.view(torch.uint8).cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n, dim", [(1, 1), (1, 768), (3, 127), (5, 128), (7, 129), (4, 300), (33, 513), (2, 1000), (9, 2052),
                                    (300, 64)])
def test_write_is_the_definition(n, dim, dtype):
    import torch

    x = torch.from_numpy(rows_of(n, dim, n * 1000 + dim)).cuda().to(_dtype(dtype))
    codes, scales = vx.fp8_empty(n, dim)
    codes.view(torch.uint8).fill_(0xAA)
    vx.fp8_write_device(x, codes, scales)
    c, s = encode(x.float().cpu().numpy())
    assert np.array_equal(scales.cpu().numpy(), s)
    assert np.array_equal(_bytes(codes), c)


@pytest.mark.gpu
def test_write_of_every_rounding_case():
    """Ties between neighbouring codes, values on either side of them, the largest value's neighbours, the
    smallest codes, zeros of both signs and scales at their limits."""
    import torch

    grid = VALUES[:127]
    mid = (grid[1:] + grid[:-1]) / 2
    v = np.concatenate([grid, mid, np.nextafter(mid.astype(np.float32), np.float32(np.inf)),
                        np.nextafter(mid.astype(np.float32), np.float32(0)), [0.0, -0.0, 1e-30]])
    v = np.concatenate([v, -v]).astype(np.float32)
    rows = []
    for e in (-120, -60, -8, 0, 1, 40, 119):  # 448 2^119 is below fp32's largest value
        for at in range(0, len(v), BLOCK - 1):
            block = np.zeros(BLOCK, np.float32)
            part = v[at : at + BLOCK - 1]
            block[: len(part)] = part
            block[-1] = 448.0
            rows.append(block.astype(np.float64) * 2.0 ** e)
    x = np.array(rows)
    assert np.abs(x).max() <= np.finfo(np.float32).max
    edge = np.zeros((6, BLOCK))
    edge[0, 3] = np.finfo(np.float32).max
    edge[1, 3] = np.finfo(np.float32).smallest_subnormal
    edge[2, 3] = 448 * 2.0 ** -127
    edge[3, 3] = np.nextafter(np.float32(448), np.float32(1000))
    edge[4, :4] = [np.finfo(np.float32).tiny, -np.finfo(np.float32).tiny, 1e-41, -1e-42]
    x = np.concatenate([x, edge]).astype(np.float32)
    codes, scales = vx.fp8_empty(len(x), BLOCK)
    vx.fp8_write_device(torch.from_numpy(x).cuda(), codes, scales)
    c, s = encode(x)
    assert np.array_equal(scales.cpu().numpy(), s)
    assert np.array_equal(_bytes(codes), c)


@pytest.mark.gpu
def test_blocks_with_nan_or_infinity_are_nan():
    import torch

    x = rows_of(6, 300, 1)
    x[1, 5], x[2, 128], x[3, 299], x[4, 7] = np.nan, np.inf, -np.inf, -np.nan
    codes, scales = vx.fp8_empty(6, 300)
    vx.fp8_write_device(torch.from_numpy(x).cuda(), codes, scales)
    c, s = encode(x)
    assert np.array_equal(scales.cpu().numpy(), s) and np.array_equal(_bytes(codes), c)
    got = vx.fp8_read_device(codes, scales, 300).cpu().numpy()
    assert np.array_equal(got, decode(c, s)[:, :300].astype(np.float32), equal_nan=True)
    assert np.isnan(got[2, 128:256]).all() and np.isfinite(got[2, :128]).all()
    sc = vx.fp8_scores_device(torch.from_numpy(rows_of(3, 300, 2)).cuda(), codes, scales).cpu().numpy()
    assert np.isnan(sc[:, 1:5]).all() and np.isfinite(sc[:, [0, 5]]).all()
    back = vx.fp8_scores_device(torch.from_numpy(x).cuda(), *_store(rows_of(3, 300, 2))).cpu().numpy()
    assert np.isnan(back[1:5]).all() and np.isfinite(back[[0, 5]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int32", "int64"])
@pytest.mark.parametrize("n", [1, 2, 37, 257, 512, 513, 5000, 8192, 8193, 20000])
def test_write_to_slots(n, kind):
    """Scattered, repeated and skipped slots: the last row of a slot is kept, other slots stay."""
    import torch

    r = np.random.default_rng(n)
    capacity, dim = 2 * n + 3, 200
    x = rows_of(n, dim, n + 5)
    slots = r.integers(-2, capacity + 2, n)
    if n > 2:
        slots[n // 2] = slots[0]
        slots[-1] = slots[1]
        slots[2] = 1 << 30
    before_c = r.integers(0, 127, (capacity, 256)).astype(np.uint8)
    before_s = r.integers(1, 200, (capacity, 4)).astype(np.uint8)
    codes, scales = torch.from_numpy(before_c.copy()).cuda(), torch.from_numpy(before_s.copy()).cuda()
    for _ in range(3):  # the same result each time
        vx.fp8_write_device(torch.from_numpy(x).cuda(), codes, scales, slots=torch.from_numpy(slots).cuda().to(_dtype(kind)))
    c, s = encode(x)
    for i, slot in enumerate(slots):
        if 0 <= slot < capacity:
            before_c[slot], before_s[slot] = c[i], s[i]
    assert np.array_equal(_bytes(codes), before_c)
    assert np.array_equal(scales.cpu().numpy(), before_s)


@pytest.mark.gpu
def test_every_row_to_one_slot():
    import torch

    x = rows_of(9000, 130, 9)
    for n in (200, 1000, 3000, 9000):
        codes, scales = vx.fp8_empty(5, 130)
        vx.fp8_write_device(torch.from_numpy(x[:n]).cuda(), codes, scales, slots=torch.full((n,), 2, device="cuda"))
        c, s = encode(x[n - 1 : n])
        assert np.array_equal(_bytes(codes)[2], c[0]) and np.array_equal(scales.cpu().numpy()[2], s[0])
        assert not _bytes(codes)[[0, 1, 3, 4]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("view", ["shifted", "columns", "transposed", "broadcast", "rows"])
def test_strided_rows(view, dtype):
    import torch

    base = torch.from_numpy(rows_of(40, 411, 3)).cuda().to(_dtype(dtype))
    x = {"shifted": base.reshape(-1)[1:].narrow(0, 0, 12 * 400).view(12, 400), "columns": base[:, 3:303],
         "transposed": base.t()[:30], "broadcast": base[:1].expand(9, 411), "rows": base[5::7]}[view]
    n, dim = x.shape
    codes, scales = vx.fp8_empty(n + 2, dim)
    vx.fp8_write_device(x, codes, scales, first=2)
    c, s = encode(x.float().cpu().numpy())
    assert np.array_equal(_bytes(codes)[2:], c) and np.array_equal(scales.cpu().numpy()[2:], s)
    assert not _bytes(codes)[:2].any()
    got = vx.fp8_scores_device(x, codes[2:], scales[2:]).cpu().numpy()
    d = decode(c, s)
    assert (np.abs(got - d @ d.T) <= bound(d, d, "float32")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n, dim", [(1, 1), (6, 127), (5, 300), (9, 768), (4, 2052)])
def test_read_back(n, dim, dtype):
    import torch

    c, s = encode(rows_of(n, dim, dim))
    codes, scales = torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda()
    want = torch.from_numpy(decode(c, s)[:, :dim].astype(np.float32)).to(_dtype(dtype))
    assert torch.equal(vx.fp8_read_device(codes, scales, dim, dtype=_dtype(dtype)).cpu(), want)
    assert torch.equal(vx.fp8_read_device(codes, scales, dim, first=n - 1, dtype=_dtype(dtype)).cpu(), want[-1:])
    slots = torch.tensor([n - 1, -1, 0, n, 0, 2 ** 30, n - 1], device="cuda")
    for kind in (torch.int32, torch.int64):
        got = vx.fp8_read_device(codes, scales, dim, slots=slots.to(kind), dtype=_dtype(dtype)).cpu()
        for i, slot in enumerate(slots.tolist()):
            assert torch.equal(got[i], want[slot] if 0 <= slot < n else torch.zeros(dim, dtype=_dtype(dtype)))
    wide = torch.full((n, dim + 5), 7.0, dtype=_dtype(dtype), device="cuda")
    vx.fp8_read_device(codes, scales, dim, out=wide[:, 2 : dim + 2])
    assert torch.equal(wide[:, 2 : dim + 2].cpu(), want)
    assert (wide[:, :2] == 7).all() and (wide[:, dim + 2 :] == 7).all()


@pytest.mark.gpu
def test_every_code_and_scale_reads_back():
    import torch

    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    scales = np.zeros((256, 4), np.uint8)
    scales[:, 0] = scales[:, 1] = np.arange(256)
    got = vx.fp8_read_device(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), 256).cpu().numpy()
    with np.errstate(over="ignore"):
        want = decode(codes, scales).astype(np.float32)
    assert np.array_equal(got, want, equal_nan=True)


# ---------------------------------------------------------------- on the GPU: products
@pytest.mark.gpu
@pytest.mark.parametrize("nq, n, dim", [(1, 1, 1), (1, 255, 100), (16, 256, 128), (17, 257, 129), (31, 300, 512), (33, 1000, 513),
                                        (224, 513, 640), (225, 700, 768), (100, 40000, 64), (500, 1111, 1500), (3, 70000, 200),
                                        (1000, 300, 2048), (64, 20000, 256), (37, 5003, 300), (1, 600, 16384)])
@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
def test_scores(nq, n, dim, out):
    import torch

    spread = 1.0 if out == "float16" else 3.0
    q, x = rows_of(nq, dim, nq, spread), rows_of(n, dim, n + 1, spread)
    codes, scales = vx.fp8_empty(n, dim)
    vx.fp8_write_device(torch.from_numpy(x).cuda(), codes, scales)
    dq, dr = decode(*encode(q)), decode(_bytes(codes), scales.cpu().numpy())
    want, tol = dq @ dr.T, bound(dq, dr, out)
    for queries in ("float32", "float16", "bfloat16", "stored"):
        if queries == "stored":
            qc, qs = _store(q)
            got = vx.fp8_scores_device(qc, codes, scales, query_scales=qs, dtype=_dtype(out))
        else:
            tq = torch.from_numpy(q).cuda().to(_dtype(queries))
            if queries != "float32":
                dt = decode(*encode(tq.float().cpu().numpy()))
                want, tol = dt @ dr.T, bound(dt, dr, out)
            got = vx.fp8_scores_device(tq, codes, scales, dtype=_dtype(out))
            if queries == "float32":
                assert torch.equal(got, vx.fp8_scores_device(tq, codes, scales, dtype=_dtype(out)))
        if queries == "stored":
            want, tol = dq @ dr.T, bound(dq, dr, out)
        assert got.shape == (nq, n) and got.dtype == _dtype(out)
        err = np.abs(got.float().cpu().numpy().astype(np.float64) - want)
        assert (err <= tol).all(), (queries, err.max(), np.argwhere(err > tol)[:5])


@pytest.mark.gpu
def test_scores_apply_each_block_scale():
    """One element per block, every block of every row and query with its own scale: the sums are exact."""
    import torch

    r = np.random.default_rng(4)
    nq, n, nb = 230, 600, 9
    x, q = np.zeros((n, nb * BLOCK)), np.zeros((nq, nb * BLOCK))
    for b in range(nb):
        x[:, b * BLOCK + 3 * b] = 2.0 ** r.integers(-6, 6, n)
        q[:, b * BLOCK + 3 * b] = 2.0 ** r.integers(-6, 6, nq)
    got = vx.fp8_scores_device(torch.from_numpy(q.astype(np.float32)).cuda(), *_store(x)).cpu().numpy()
    assert np.array_equal(got.astype(np.float64), q @ x.T)


@pytest.mark.gpu
def test_scores_into_a_larger_tensor():
    import torch

    q, x = rows_of(21, 100, 1), rows_of(333, 100, 2)
    codes, scales = _store(x)
    dq, dr = decode(*encode(q)), decode(_bytes(codes), scales.cpu().numpy())
    for off in (0, 1, 3):
        for name in ("float32", "bfloat16"):
            wide = torch.full((21, 340), -5.0, dtype=_dtype(name), device="cuda")
            vx.fp8_scores_device(torch.from_numpy(q).cuda(), codes, scales, out=wide[:, off : off + 333])
            got = wide.float().cpu().numpy().astype(np.float64)
            assert (np.abs(got[:, off : off + 333] - dq @ dr.T) <= bound(dq, dr, name)).all()
            assert (got[:, :off] == -5).all() and (got[:, off + 333 :] == -5).all()


def _grouped_want(q, x, qo, ro, max_rows, fill):
    want = np.full((len(q), max_rows), fill)
    tol = np.zeros((len(q), max_rows))
    for g in range(len(qo) - 1):
        a, b = max(0, min(qo[g], len(q))), max(0, min(qo[g + 1], len(q)))
        c, d = max(0, min(ro[g], len(x))), max(0, min(ro[g + 1], len(x)))
        d = min(d, c + max_rows)
        if a < b and c < d:
            want[a:b, : d - c] = q[a:b] @ x[c:d].T
            tol[a:b, : d - c] = bound(q[a:b], x[c:d], "float32")
    return want, tol


@pytest.mark.gpu
@pytest.mark.parametrize("groups, nq, n, dim, seed", [(1, 5, 40, 100, 0), (3, 17, 900, 128, 1), (40, 300, 5000, 200, 2),
                                                      (7, 2000, 3000, 768, 3), (1500, 400, 2000, 64, 4), (5, 1, 100, 640, 5)])
def test_grouped(groups, nq, n, dim, seed):
    """Ragged groups, many of them empty on one side or both."""
    import torch

    r = np.random.default_rng(seed)
    q, x = rows_of(nq, dim, seed + 10), rows_of(n, dim, seed + 20)
    qo = np.sort(np.concatenate([[0, nq], r.integers(0, nq + 1, groups - 1)]))
    ro = np.sort(np.concatenate([[0, n], r.integers(0, n + 1, groups - 1)]))
    if groups > 4:
        qo[2], ro[3] = qo[1], ro[2]
    codes, scales = _store(x)
    dq, dr = decode(*encode(q)), decode(_bytes(codes), scales.cpu().numpy())
    width = int((ro[1:] - ro[:-1]).max())
    tqo, tro = torch.from_numpy(qo).cuda(), torch.from_numpy(ro).cuda()
    for max_rows in {width, max(1, width // 2), width + 3}:
        want, tol = _grouped_want(dq, dr, qo, ro, max_rows, -3.0)
        for stored in (False, True):
            out = torch.full((nq, max_rows), -3.0, device="cuda")
            if stored:
                qc, qs = _store(q)
                got = vx.fp8_scores_grouped_device(qc, tqo, codes, scales, tro, query_scales=qs, out=out)
            else:
                got = vx.fp8_scores_grouped_device(torch.from_numpy(q).cuda(), tqo, codes, scales, tro, out=out)
            assert got is out
            err = np.abs(out.cpu().numpy().astype(np.float64) - want)
            assert (err <= tol).all(), (stored, err.max(), np.argwhere(err > tol)[:5])
    fresh = vx.fp8_scores_grouped_device(torch.from_numpy(q).cuda(), tqo, codes, scales, tro, max_rows=width,
                                         dtype=torch.bfloat16)
    want, _ = _grouped_want(dq, dr, qo, ro, width, 0.0)
    assert fresh.dtype == torch.bfloat16 and not fresh.float().cpu().numpy()[want == 0.0].any()


@pytest.mark.gpu
def test_grouped_with_offsets_out_of_range():
    """Offsets past the operands, negative or descending: clamped, the group empty where its end comes first."""
    import torch

    q, x = rows_of(30, 100, 1), rows_of(700, 100, 2)
    codes, scales = _store(x)
    dq, dr = decode(*encode(q)), decode(_bytes(codes), scales.cpu().numpy())
    qo, ro = [-5, 4, 10, 8, 25, 1 << 40], [-(1 << 50), 100, 50, 400, 600, 1 << 60]
    # query ranges: [0,4) [4,10) none [8,25) [25,30); row ranges: [0,100) none [50,400) [400,600) [600,700)
    want, tol = _grouped_want(dq, dr, qo, ro, 350, 9.0)
    out = torch.full((30, 350), 9.0, device="cuda")
    vx.fp8_scores_grouped_device(torch.from_numpy(q).cuda(), torch.tensor(qo, device="cuda"), codes, scales,
                                 torch.tensor(ro, device="cuda"), out=out)
    assert (np.abs(out.cpu().numpy() - want) <= tol).all()


@pytest.mark.gpu
def test_nothing_to_do():
    import torch

    codes, scales = vx.fp8_empty(0, 100)
    q = torch.randn(3, 100, device="cuda")
    assert vx.fp8_scores_device(q, codes, scales).shape == (3, 0)
    assert vx.fp8_read_device(codes, scales, 100).shape == (0, 100)
    assert (vx.fp8_read_device(codes, scales, 100, slots=torch.tensor([-1, 0], device="cuda")) == 0).all()
    vx.fp8_write_device(q, codes, scales, slots=torch.tensor([0, 1, 2], device="cuda"))
    codes, scales = vx.fp8_empty(5, 100)
    vx.fp8_write_device(q[:0], codes, scales)
    vx.fp8_write_device(q[:0], codes, scales, slots=torch.zeros(0, dtype=torch.int64, device="cuda"))
    none = torch.zeros(1, dtype=torch.int64, device="cuda")
    assert (vx.fp8_scores_grouped_device(q, none, codes, scales, none, max_rows=4) == 0).all()
    zero = torch.zeros(3, dtype=torch.int64, device="cuda")
    assert (vx.fp8_scores_grouped_device(q, zero, codes, scales, zero, max_rows=4) == 0).all()
    assert vx.fp8_scores_grouped_device(q[:0], zero, codes, scales, zero, max_rows=4).shape == (0, 4)
    with pytest.raises(vx.IllegalArgumentException, match="empty"):
        vx.fp8_scores_device(q[:0], codes, scales)
    vx.fp8_check()


@pytest.mark.gpu
def test_refusals_of_tensors():
    import torch

    codes, scales = vx.fp8_empty(50, 100)
    q = torch.randn(3, 100, device="cuda")
    off = torch.tensor([0, 3], device="cuda")
    bad = vx.IllegalArgumentException
    for call in (lambda: vx.fp8_write_device(q, codes, scales, first=48), lambda: vx.fp8_write_device(q.double(), codes, scales),
                 lambda: vx.fp8_write_device(torch.zeros(3, 129, device="cuda"), codes, scales),
                 lambda: vx.fp8_write_device(q[0], codes, scales), lambda: vx.fp8_write_device(q.cpu(), codes, scales),
                 lambda: vx.fp8_write_device(q, codes[::2], scales[::2]),
                 lambda: vx.fp8_write_device(q, codes, scales, slots=off),
                 lambda: vx.fp8_write_device(q, codes, scales, slots=torch.zeros(3, device="cuda")),
                 lambda: vx.fp8_write_device(q, codes, scales, slots=torch.zeros(3, dtype=torch.int64)),
                 lambda: vx.fp8_read_device(codes, scales, 200), lambda: vx.fp8_read_device(codes, scales, 100, count=51),
                 lambda: vx.fp8_read_device(codes, scales, 100, first=51), lambda: vx.fp8_read_device(codes, scales, 100, first=-1, count=2),
                 lambda: vx.fp8_read_device(codes, scales, 100, dtype=torch.int8),
                 lambda: vx.fp8_read_device(codes, scales, 100, slots=off, count=3),
                 lambda: vx.fp8_read_device(codes, scales, 100, out=torch.zeros(100, 50, device="cuda").t()),
                 lambda: vx.fp8_scores_device(torch.zeros(3, 300, device="cuda"), codes, scales),
                 lambda: vx.fp8_scores_device(q, codes, scales, out=torch.zeros(3, 49, device="cuda")),
                 lambda: vx.fp8_scores_device(q, codes, scales, out=torch.zeros(1, 50, device="cuda").expand(3, 50)),
                 lambda: vx.fp8_scores_device(q, codes, scales, out=torch.zeros(3, 50)),
                 lambda: vx.fp8_scores_device(q, codes, scales, dtype=torch.float64),
                 lambda: vx.fp8_scores_device(codes, codes, scales, query_scales=scales[:49]),
                 lambda: vx.fp8_scores_grouped_device(q, off.int(), codes, scales, off, max_rows=50),
                 lambda: vx.fp8_scores_grouped_device(q, off, codes, scales, off[:1], max_rows=50),
                 lambda: vx.fp8_scores_grouped_device(q, off, codes, scales, off),
                 lambda: vx.fp8_scores_grouped_device(q, off, codes, scales, off.cpu(), max_rows=50)):
        with pytest.raises(bad):
            call()


@pytest.mark.gpu
def test_scores_of_extreme_scales():
    """Scales whose product is ordinary, leaves fp32 upwards (infinity) or downwards (at most its smallest
    normal number off)."""
    import torch

    q, x = rows_of(40, 256, 1, 0.5).astype(np.float64), rows_of(300, 256, 2, 0.5).astype(np.float64)
    with np.errstate(over="ignore"):
        for eq, er in ((100, -100), (-110, 110), (-60, -70), (-100, -100), (70, 70)):
            a, b = (q * 2.0 ** eq).astype(np.float32), (x * 2.0 ** er).astype(np.float32)
            codes, scales = _store(b)
            got = vx.fp8_scores_device(torch.from_numpy(a).cuda(), codes, scales).cpu().numpy().astype(np.float64)
            dq, dr = decode(*encode(a)), decode(_bytes(codes), scales.cpu().numpy())
            want, tol = dq @ dr.T, bound(dq, dr, "float32") + 2.0 ** -126
            # where single terms pass fp32's range (2^140 here), a partial sum is infinite before the last term
            # is in, with that partial sum's sign and not the result's: only "not finite" follows
            huge = np.abs(want) > 2.0 ** 129
            assert not np.isfinite(got[huge]).any()
            fine = np.abs(want) + tol < 2.0 ** 127
            assert (np.abs(got - want) <= tol)[fine].all()
            assert fine.all() or eq + er > 100


@pytest.mark.gpu
def test_groups_that_share_rows():
    """The same rows scored for several groups, and a group with the same offsets twice."""
    import torch

    q, x = rows_of(50, 200, 1), rows_of(900, 200, 2)
    codes, scales = _store(x)
    dq, dr = decode(*encode(q)), decode(_bytes(codes), scales.cpu().numpy())
    want = dq @ dr.T
    tol = bound(dq, dr, "float32")
    # 10 queries x rows 0-600, none, 20 x none (descending), 20 x 300-900: offsets ascend only per operand's rule
    qo = torch.tensor([0, 10, 10, 30, 50], device="cuda")
    ro = torch.tensor([0, 600, 600, 300, 900], device="cuda")
    out = torch.full((50, 600), -1.0, device="cuda")
    vx.fp8_scores_grouped_device(torch.from_numpy(q).cuda(), qo, codes, scales, ro, out=out)
    got = out.cpu().numpy().astype(np.float64)
    assert (np.abs(got[:10] - want[:10, :600]) <= tol[:10, :600]).all()
    assert (got[10:30] == -1).all()
    assert (np.abs(got[30:] - want[30:, 300:900]) <= tol[30:, 300:900]).all()


@pytest.mark.gpu
def test_store_past_32_bits():
    """Slots whose codes lie past 2^32 bytes, written, read back and scored."""
    import torch

    if torch.cuda.get_device_properties(0).total_memory < 32 << 30:
        pytest.skip("needs 32 GB")
    capacity, dim = 4_400_000, 1000
    codes, scales = vx.fp8_empty(capacity, dim)
    x = rows_of(700, dim, 1)
    slots = torch.cat([torch.arange(capacity - 600, capacity), torch.arange(100)]).cuda()
    vx.fp8_write_device(torch.from_numpy(x).cuda(), codes, scales, slots=slots)
    c, s = encode(x)
    assert np.array_equal(_bytes(codes[-600:]), c[:600]) and np.array_equal(scales[-600:].cpu().numpy(), s[:600])
    back = vx.fp8_read_device(codes, scales, dim, slots=slots)
    assert np.array_equal(back.cpu().numpy(), decode(c, s)[:, :dim].astype(np.float32))
    assert torch.equal(vx.fp8_read_device(codes, scales, dim, first=capacity - 600), back[:600])
    q = rows_of(3, dim, 2)
    got = vx.fp8_scores_device(torch.from_numpy(q).cuda(), codes, scales)
    dq, dr = decode(*encode(q)), decode(c, s)
    assert (np.abs(got[:, slots].cpu().numpy() - dq @ dr.T) <= bound(dq, dr, "float32")).all()
    assert not got[:, 100:-600].any()
    ro = torch.tensor([0, 100, capacity - 600, capacity], device="cuda")
    out = torch.zeros(3, 600, device="cuda")
    vx.fp8_scores_grouped_device(torch.from_numpy(q).cuda(), torch.tensor([0, 1, 1, 3], device="cuda"), codes, scales, ro,
                                 out=out)
    assert torch.equal(out[0, :100], got[0, :100]) and torch.equal(out[1:], got[1:, -600:])


@pytest.mark.gpu
def test_results_past_32_bits():
    """A score matrix of more than 2^31 results."""
    import torch

    if torch.cuda.get_device_properties(0).total_memory < 32 << 30:
        pytest.skip("needs 32 GB")
    q, x = rows_of(47000, 128, 1, 1.0), rows_of(46000, 128, 2, 1.0)
    qc, qs, codes, scales = *vx.fp8_empty(47000, 128), *vx.fp8_empty(46000, 128)
    vx.fp8_write_device(torch.from_numpy(q).cuda(), qc, qs)
    vx.fp8_write_device(torch.from_numpy(x).cuda(), codes, scales)
    got = vx.fp8_scores_device(qc, codes, scales, query_scales=qs, dtype=torch.bfloat16)
    assert got.numel() > 2 ** 31
    for at in (slice(0, 50), slice(23400, 23450), slice(46950, 47000)):
        part = vx.fp8_scores_device(qc[at], codes, scales, query_scales=qs[at], dtype=torch.bfloat16)
        assert torch.equal(got[at], part)
    at = slice(46990, 47000)
    dq, dr = decode(_bytes(qc[at]), qs[at].cpu().numpy()), decode(_bytes(codes), scales.cpu().numpy())
    assert (np.abs(got[at].float().cpu().numpy() - dq @ dr.T) <= bound(dq, dr, "bfloat16")).all()


# ---------------------------------------------------------------- streams, graphs, the operators together
@pytest.mark.gpu
def test_other_stream_and_graph():
    """Two captured graphs whose scratch may share memory, replayed in turn on changed inputs, and calls on a
    stream other than the current one."""
    import torch

    n, nq, dim = 3000, 70, 300
    x = torch.from_numpy(rows_of(n, dim, 1)).cuda()
    q1, q2 = (torch.from_numpy(rows_of(nq, dim, s)).cuda() for s in (2, 3))
    slots = torch.randperm(n, device="cuda")
    codes, scales = vx.fp8_empty(n, dim)
    qo = torch.tensor([0, 10, 40, 70], device="cuda")
    ro = torch.tensor([0, 1200, 1300, 3000], device="cuda")
    outs = [torch.zeros(nq, n, device="cuda"), torch.zeros(nq, 1700, device="cuda")]

    def one():
        vx.fp8_write_device(x, codes, scales, slots=slots)
        vx.fp8_scores_device(q1, codes, scales, out=outs[0])

    def two():
        vx.fp8_scores_grouped_device(q2, qo, codes, scales, ro, out=outs[1])

    one()
    two()
    torch.cuda.synchronize()
    graphs = []
    for f in (one, two):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            f()
        graphs.append(g)
    for seed in (11, 12):
        x.copy_(torch.from_numpy(rows_of(n, dim, seed)))
        q1.copy_(torch.from_numpy(rows_of(nq, dim, seed + 1)))
        q2.copy_(torch.from_numpy(rows_of(nq, dim, seed + 2)))
        for o in outs:
            o.fill_(-1.0)
        for g in graphs + graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        c2, s2 = vx.fp8_empty(n, dim)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        vx.fp8_write_device(x, c2, s2, slots=slots, stream=side.cuda_stream)
        a = vx.fp8_scores_device(q1, c2, s2, stream=side.cuda_stream)
        b = vx.fp8_scores_grouped_device(q2, qo, c2, s2, ro, max_rows=1700, stream=side.cuda_stream)
        side.synchronize()
        assert torch.equal(codes.view(torch.uint8), c2.view(torch.uint8)) and torch.equal(scales, s2)
        assert torch.equal(outs[0], a)
        assert torch.equal(torch.where(b == 0, b, outs[1]), b)
        dq, dr = decode(*encode(q1.cpu().numpy())), decode(_bytes(codes), scales.cpu().numpy())
        assert (np.abs(a.cpu().numpy() - dq @ dr.T) <= bound(dq, dr, "float32")).all()


CAPTURED_FIRST = """
import torch, vectors_b200 as vx
x, q = torch.randn(3000, 300, device="cuda"), torch.randn(70, 300, device="cuda")
codes, scales = vx.fp8_empty(4000, 300)
slots = torch.randperm(4000, device="cuda")[:3000]
out, few = torch.zeros(70, 4000, device="cuda"), torch.zeros(2, 4000, device="cuda")
grouped = torch.zeros(70, 4000, device="cuda")
qo, ro = torch.tensor([0, 30, 70], device="cuda"), torch.tensor([0, 1000, 4000], device="cuda")
back = torch.zeros(3000, 300, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):  # the library's first calls in this process
    vx.fp8_write_device(x, codes, scales, slots=slots)
    vx.fp8_scores_device(q, codes, scales, out=out)
    vx.fp8_scores_device(q[:2], codes, scales, out=few)
    vx.fp8_scores_grouped_device(q, qo, codes, scales, ro, out=grouped)
    vx.fp8_read_device(codes, scales, 300, slots=slots, out=back)
g.replay()
torch.cuda.synchronize()
c, s = vx.fp8_empty(4000, 300)
vx.fp8_write_device(x, c, s, slots=slots)
want = vx.fp8_scores_device(q, c, s)
assert torch.equal(codes.view(torch.uint8), c.view(torch.uint8)) and torch.equal(out, want)
assert torch.equal(few, want[:2])
assert torch.equal(grouped[:30, :1000], want[:30, :1000]) and torch.equal(grouped[30:, :3000], want[30:, 1000:])
assert torch.equal(back, vx.fp8_read_device(c, s, 300, slots=slots))
vx.fp8_check()
print("captured first: ok")
"""


@pytest.mark.gpu
def test_first_calls_inside_a_capture():
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured first: ok" in run.stdout, run.stdout + run.stderr


@pytest.mark.gpu
def test_results_of_a_pair_do_not_depend_on_the_call():
    """The same query and row give the same bits as one of many queries, alone, from a stored copy, and in a
    group: each result is one sum over dimensions in one order."""
    import torch

    x, q = torch.from_numpy(rows_of(5000, 700, 1)).cuda(), torch.from_numpy(rows_of(300, 700, 2)).cuda()
    codes, scales = vx.fp8_empty(5000, 700)
    vx.fp8_write_device(x, codes, scales)
    many = vx.fp8_scores_device(q, codes, scales)
    qc, qs = vx.fp8_empty(300, 700)
    vx.fp8_write_device(q, qc, qs)
    assert torch.equal(vx.fp8_scores_device(qc, codes, scales, query_scales=qs), many)
    for n in (1, 20, 40, 100):
        assert torch.equal(vx.fp8_scores_device(q[:n], codes, scales), many[:n])
    assert torch.equal(vx.fp8_scores_device(q, codes[17:3001], scales[17:3001]), many[:, 17:3001])
    off = torch.tensor([0, 7, 300], device="cuda")
    rows = torch.tensor([0, 1234, 5000], device="cuda")
    grouped = vx.fp8_scores_grouped_device(q, off, codes, scales, rows, max_rows=4000)
    assert torch.equal(grouped[:7, :1234], many[:7, :1234]) and torch.equal(grouped[7:, :3766], many[7:, 1234:])


@pytest.mark.gpu
def test_two_threads_at_once():
    import threading

    import torch

    x, q = rows_of(4000, 256, 1), [rows_of(50, 256, s) for s in range(4)]
    codes, scales = _store(x)
    want = [vx.fp8_scores_device(torch.from_numpy(a).cuda(), codes, scales).cpu() for a in q]
    got = [None] * 4

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                got[i] = vx.fp8_scores_device(torch.from_numpy(q[i]).cuda(), codes, scales)
        st.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        assert torch.equal(got[i].cpu(), want[i])


@pytest.mark.gpu
def test_together_behind_ivf_routing():
    """The operators as a collection uses them: rows ingested list by list in two batches, queries routed by
    the IVF index, each list's queries scored against its rows, the best candidates read back and re-scored;
    the neighbours are those of the exact IVF search except where 8-bit scores cannot tell them apart."""
    import torch

    r = np.random.default_rng(0)
    n, dim, nlist, nq, k, probes = 6000, 96, 24, 40, 10, 4
    centers = r.standard_normal((nlist, dim)).astype(np.float32) * 2
    x = (centers[r.integers(0, nlist, n)] + r.standard_normal((n, dim))).astype(np.float32)
    assign = ((x[:, None, :] - centers[None]) ** 2).sum(2).argmin(1)
    order = np.argsort(assign, kind="stable").astype(np.int32)
    off = np.concatenate([[0], np.cumsum(np.bincount(assign, minlength=nlist))]).astype(np.int64)
    q = (x[r.integers(0, n, nq)] + 0.3 * r.standard_normal((nq, dim))).astype(np.float32)

    ivf = vx.IvfFlatAdapter(nprobe=probes)
    ivf.build_prebuilt(centers, off, order, x, vx.SimilarityFunction.DOT_PRODUCT)
    tq = torch.from_numpy(q).cuda()
    lists = ivf.route_device(tq, probes)
    exact_ids, _, _ = ivf.ivf_search_device(tq, k, probes)

    # store: slot = the row's place in its list; two ingest batches in arrival order
    place = np.empty(n, np.int64)
    place[order] = np.arange(n)
    codes, scales = vx.fp8_empty(n, dim)
    half = n // 2
    for a, b in ((0, half), (half, n)):
        vx.fp8_write_device(torch.from_numpy(x[a:b]).cuda(), codes, scales, slots=torch.from_numpy(place[a:b]).cuda())

    pair_list = lists.long().reshape(-1)
    by_list = torch.argsort(pair_list, stable=True)
    qo = torch.searchsorted(pair_list[by_list], torch.arange(nlist + 1, device="cuda"))
    ro = torch.from_numpy(off).cuda()
    width = int((off[1:] - off[:-1]).max())
    out = torch.full((nq * probes, width), -torch.inf, device="cuda")
    vx.fp8_scores_grouped_device(tq[by_list // probes], qo, codes, scales, ro, out=out)
    per_query = torch.empty_like(out)
    per_query[by_list] = out
    per_query = per_query.view(nq, probes * width)
    cand = per_query.topk(4 * k, dim=1).indices
    slots = ro[lists.long().gather(1, cand // width)] + cand % width
    rows = vx.fp8_read_device(codes, scales, dim, slots=slots.reshape(-1)).view(nq, 4 * k, dim)
    # the read-back rows rank as the scores did (same stored rows, queries unquantised)
    err = (rows - torch.from_numpy(x).cuda()[torch.from_numpy(order.astype(np.int64)).cuda()[slots]]).norm(dim=2)
    assert (err <= 2.0 ** -4 * rows.norm(dim=2) * 1.2).all()
    full = vx.fp8_scores_device(tq, codes, scales)
    # both products of a pair sum the same terms: at most dim 2^-23 |q| |r| each from the exact sum
    tol = 2 * 128 * 2.0 ** -23 * 1.1 * tq.norm(dim=1)[:, None] * rows.norm(dim=2).amax(1)[:, None]
    assert ((full.gather(1, slots) - per_query.gather(1, cand)).abs() <= tol).all()
    # an exact neighbour is among the candidates, or its 8-bit score is below theirs
    mine = torch.from_numpy(place).cuda()[exact_ids.long()]
    found = (mine[:, :, None] == slots[:, None, :]).any(2)
    least = per_query.gather(1, cand).amin(1, keepdim=True)
    assert (found | (full.gather(1, mine) <= least + tol)).all()
    ivf.close()
