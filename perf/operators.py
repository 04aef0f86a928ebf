"""The 8-bit float row operators, measured: what a pass takes in, what it returns, and its plain form.

The operators keep rows as e4m3 codes with one power-of-two scale for each block of 128
dimensions (codes [rows][dim rounded up to 128], scale exponents [rows][blocks rounded up to 4],
a byte b standing for 2^(b - 127)):

* write   rows are quantised into given slots of the store;
* read    stored rows are brought back as floats;
* scores  the product of a query batch with every stored row;
* grouped the products of each group of queries with that group's stored rows (an inverted
          list's candidates, an expert's weights), all group sizes different.

``run`` computes them with elementary torch operations in 32 bits, or with the library's kernels
where ``own`` is true.
"""
import random

import torch

own = False

BLOCK = 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}


def blocks_of(dim):
    return -(-dim // BLOCK)


def row_bytes(dim):
    """Bytes of one stored row: its codes and its scale exponents."""
    return blocks_of(dim) * BLOCK + -(-blocks_of(dim) // 4) * 4


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one document upserted into a live collection: latency
        {"name": "write_one", "op": "write", "n": 1, "dim": 768, "type": "f32", "capacity": 4096, "slots": True},
        # an ingest batch from an embedder in bf16, scattered over free slots, some rows padding
        {"name": "write_batch", "op": "write", "n": 10007, "dim": 768, "type": "bf16", "capacity": 50000, "slots": True},
        # a collection loaded whole, rows in order
        {"name": "write_bulk", "op": "write", "n": 400000, "dim": 1024, "type": "f32", "capacity": 400000, "slots": False},
        # the candidates of ten searches with k = 100 brought back for a second look
        {"name": "read_window", "op": "read", "n": 1000, "dim": 768, "type": "f32", "capacity": 100000, "slots": True},
        # a third of a large collection re-read in another order, of an odd dimension
        {"name": "read_bulk", "op": "read", "n": 300000, "dim": 1000, "type": "f16", "capacity": 400000, "slots": True},
        # one query against a collection: reads the rows once, latency counts
        {"name": "scores_one", "op": "scores", "nq": 1, "n": 100000, "dim": 768, "type": "f32", "out": "f32"},
        # a small odd batch over a small collection of an odd dimension
        {"name": "scores_odd", "op": "scores", "nq": 37, "n": 5003, "dim": 300, "type": "f16", "out": "f32"},
        # the benchmark's smallest configuration as a full score matrix
        {"name": "scores_batch", "op": "scores", "nq": 1000, "n": 100000, "dim": 768, "type": "f32", "out": "f32"},
        # stored rows against stored rows (near-duplicates, assignment to centroids)
        {"name": "scores_join", "op": "scores", "nq": 8192, "n": 65536, "dim": 1024, "type": "e4m3", "out": "bf16"},
        # one query over the eight lists it was routed to
        {"name": "grouped_one", "op": "grouped", "groups": 8, "pairs": 8, "rows": 2500, "dim": 128, "type": "f32",
         "out": "f32", "spread": 0.5, "plan": 1},
        # a thousand queries routed to eight of 410 uneven lists
        {"name": "grouped_lists", "op": "grouped", "groups": 410, "pairs": 8000, "rows": 100000, "dim": 768, "type": "f32",
         "out": "f32", "spread": 0.6, "plan": 2},
        # a token batch over sixteen experts' weights, one matrix a group
        {"name": "grouped_experts", "op": "grouped", "groups": 16, "pairs": 16384, "rows": 32768, "dim": 1024, "type": "bf16",
         "out": "bf16", "spread": 0.0, "plan": 3},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))

    op = rng.choice(["write", "read", "scores", "grouped"])
    dim = rng.choice([log(16, 1536), 8 * log(2, 192), rng.choice([64, 128, 256, 384, 512, 768, 1000, 1024, 1536])])
    floats = ["f32", "f16", "bf16"]
    if op in ("write", "read"):
        n = log(1, 100000)
        return {"op": op, "n": n, "dim": dim, "type": rng.choice(floats), "capacity": n + log(1, 100000),
                "slots": rng.random() < 0.7}
    if op == "scores":
        return {"op": op, "nq": log(1, 2048), "n": log(64, 100000), "dim": dim, "type": rng.choice(floats + ["e4m3"]),
                "out": rng.choice(floats)}
    groups = log(1, 300)
    return {"op": op, "groups": groups, "pairs": log(1, 8000), "rows": log(groups, 40000), "dim": dim,
            "type": rng.choice(floats + ["e4m3"]), "out": rng.choice(floats), "spread": rng.choice([0.0, 0.5, 1.0]),
            "plan": rng.randrange(1 << 20)}


def offsets_of(case):
    """(query offsets, row offsets) of a grouped case, from the case alone: rows shared out evenly
    (spread 0) or by log-normal weights, the queries drawn towards the groups with more rows."""
    r = random.Random(case["plan"])
    groups, spread = case["groups"], case["spread"]

    def share(total, weights):
        out, done, seen, whole = [0], 0, 0.0, sum(weights)
        for w in weights:
            seen += w
            done = max(done, min(total, round(total * seen / whole)))
            out.append(done)
        out[-1] = total
        return out

    weights = [r.lognormvariate(0.0, spread) if spread else 1.0 for _ in range(groups)]
    rows = share(case["rows"], weights)
    if case["pairs"] == groups:
        return list(range(groups + 1)), rows
    counts = [0] * groups
    for g in r.choices(range(groups), weights=weights, k=case["pairs"]):
        counts[g] += 1
    queries = [0]
    for c in counts:
        queries.append(queries[-1] + c)
    return queries, rows


def width_of(case):
    _, rows = offsets_of(case)
    return max(b - a for a, b in zip(rows, rows[1:]))


def work(case):
    op, dim = case["op"], case["dim"]
    if op in ("write", "read"):
        n = case["n"] - (case["n"] // 100 if op == "write" and case["slots"] and case["n"] > 100 else 0)  # less the padding
        return {"bytes": n * (dim * SIZE[case["type"]] + row_bytes(dim) + (8 if case["slots"] else 0)), "flops": 0}
    queries = row_bytes(dim) if case["type"] == "e4m3" else dim * SIZE[case["type"]]
    out = SIZE[case["out"]]
    if op == "scores":
        nq, n = case["nq"], case["n"]
        return {"bytes": nq * queries + n * row_bytes(dim) + nq * n * out, "flops": 2 * nq * n * dim}
    qo, ro = offsets_of(case)
    sizes = [(qo[g + 1] - qo[g], ro[g + 1] - ro[g]) for g in range(case["groups"])]
    products = sum(m * n for m, n in sizes)
    read = sum(n for m, n in sizes if m)
    return {"bytes": case["pairs"] * queries + read * row_bytes(dim) + products * out + 16 * (case["groups"] + 1),
            "flops": 2 * products * dim}


# ---------------------------------------------------------------- inputs
def rows_like(n, dim, gen, device):
    """Embedding-like rows: a few directions shared by all, dimensions of different strength, lengths
    that differ from row to row."""
    strength = torch.exp(0.7 * torch.randn(dim, generator=gen, device=device))
    topics = torch.randn(16, dim, generator=gen, device=device)
    pick = torch.randint(0, 16, (n,), generator=gen, device=device)
    rows = torch.randn(n, dim, generator=gen, device=device)
    rows = (rows + topics[pick]) * strength
    length = torch.exp(0.3 * torch.randn(n, 1, generator=gen, device=device))
    return rows * (length / rows.norm(dim=1, keepdim=True).clamp_min(1e-20))


def prepare(case, seed):
    device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=device).manual_seed(int(seed))
    op, dim = case["op"], case["dim"]
    kp, sp = blocks_of(dim) * BLOCK, row_bytes(dim) - blocks_of(dim) * BLOCK
    state = {"op": op, "dim": dim}
    if op in ("write", "read"):
        n, capacity = case["n"], case["capacity"]
        state["slots"] = None
        if case["slots"]:
            slots = torch.randperm(capacity, generator=gen, device=device)[:n]
            if op == "write" and n > 100:  # every hundredth row of an ingest batch is padding
                slots = torch.where(torch.arange(n, device=device) % 100 == 99, torch.full_like(slots, -1), slots)
            state["slots"] = slots
        if op == "write":
            state["rows"] = rows_like(n, dim, gen, device).to(TYPES[case["type"]])
            state["codes"] = torch.zeros(capacity, kp, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
            state["scales"] = torch.zeros(capacity, sp, dtype=torch.uint8, device=device)
        else:
            state["codes"], state["scales"] = quantise(rows_like(capacity, dim, gen, device))
            state["count"], state["type"] = n, TYPES[case["type"]]
        return state
    n = case["n"] if op == "scores" else case["rows"]
    nq = case["nq"] if op == "scores" else case["pairs"]
    state["codes"], state["scales"] = quantise(rows_like(n, dim, gen, device))
    queries = rows_like(nq, dim, gen, device)
    state["query_scales"] = None
    if case["type"] == "e4m3":
        state["queries"], state["query_scales"] = quantise(queries)
    else:
        state["queries"] = queries.to(TYPES[case["type"]])
    if op == "scores":
        state["out"] = torch.zeros(nq, n, dtype=TYPES[case["out"]], device=device)
    else:
        qo, ro = offsets_of(case)
        state["query_offsets"] = torch.tensor(qo, dtype=torch.int64, device=device)
        state["row_offsets"] = torch.tensor(ro, dtype=torch.int64, device=device)
        state["most_queries"] = max(b - a for a, b in zip(qo, qo[1:]))
        state["out"] = torch.zeros(nq, width_of(case), dtype=TYPES[case["out"]], device=device)
    return state


# ---------------------------------------------------------------- the plain forms
def power(e):
    """2^e in 32 bits for whole -127 <= e <= 127, put together from its bits (exp2 may be off by a bit)."""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).int().view(torch.float32)


def quantise(x):
    """Codes and scale exponents of rows: the smallest power of two that brings a block's largest
    magnitude to at most 448, and the nearest e4m3 value (ties to even) of each scaled element."""
    n, dim = x.shape
    nb = blocks_of(dim)
    x = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - dim)).view(n, nb, BLOCK)
    top = x.abs().amax(2)
    part, exponent = torch.frexp(top)  # top = part 2^exponent, part in [0.5, 1); 448 = 0.875 2^9
    exponent = torch.where(top > 0, exponent - 9 + (part > 0.875).int(), torch.full_like(exponent, -127)).clamp_min(-127)
    codes = (x * power(-exponent)[:, :, None]).view(n, nb * BLOCK).to(torch.float8_e4m3fn)
    return codes, torch.nn.functional.pad((exponent + 127).to(torch.uint8), (0, -nb % 4))


def values(codes, scales):
    """The rows that codes and scale exponents stand for, in 32 bits, padding included."""
    n, kp = codes.shape
    scale = power(scales[:, : kp // BLOCK].int() - 127)
    return (codes.float().view(n, kp // BLOCK, BLOCK) * scale[:, :, None]).view(n, kp)


def run(state):
    op = state["op"]
    if own:
        import vectors_b200 as vx

        if op == "write":
            vx.fp8_write_device(state["rows"], state["codes"], state["scales"], slots=state["slots"])
            return {"codes": state["codes"], "scales": state["scales"]}
        if op == "read":
            return vx.fp8_read_device(state["codes"], state["scales"], state["dim"], slots=state["slots"],
                                      count=state["count"], dtype=state["type"])
        if op == "scores":
            return vx.fp8_scores_device(state["queries"], state["codes"], state["scales"],
                                        query_scales=state["query_scales"], out=state["out"])
        return vx.fp8_scores_grouped_device(state["queries"], state["query_offsets"], state["codes"], state["scales"],
                                            state["row_offsets"], query_scales=state["query_scales"], out=state["out"])
    if op == "write":
        codes, scales = quantise(state["rows"])
        slots = state["slots"]
        if slots is None:
            state["codes"].view(torch.uint8)[: len(codes)] = codes.view(torch.uint8)
            state["scales"][: len(codes)] = scales
        else:
            keep = slots >= 0
            state["codes"].view(torch.uint8)[slots[keep]] = codes.view(torch.uint8)[keep]
            state["scales"][slots[keep]] = scales[keep]
        return {"codes": state["codes"], "scales": state["scales"]}
    if op == "read":
        slots = state["slots"]
        if slots is None:
            codes, scales = state["codes"][: state["count"]], state["scales"][: state["count"]]
        else:
            codes, scales = state["codes"].view(torch.uint8)[slots].view(torch.float8_e4m3fn), state["scales"][slots]
        return values(codes, scales)[:, : state["dim"]].to(state["type"])
    encoded = (state["queries"], state["query_scales"]) if state["query_scales"] is not None else quantise(state["queries"])
    queries, rows, out = values(*encoded), values(state["codes"], state["scales"]), state["out"]
    if op == "scores":
        out.copy_(queries @ rows.T)
        return out
    # every group padded to the largest, one batched product, and each query's own columns taken
    qo, ro = state["query_offsets"], state["row_offsets"]
    groups, width, most = len(qo) - 1, out.shape[1], state["most_queries"]
    at = qo[:-1, None] + torch.arange(most, device=qo.device)
    left = queries[at.clamp_max(len(queries) - 1)]
    to = ro[:-1, None] + torch.arange(width, device=ro.device)
    right = rows[to.clamp_max(len(rows) - 1)]
    products = torch.bmm(left, right.transpose(1, 2)).view(groups * most, width)
    pair = torch.arange(len(queries), device=qo.device)
    group = torch.searchsorted(qo, pair, right=True) - 1
    valid = torch.arange(width, device=qo.device) < (ro[1:] - ro[:-1])[group][:, None]
    mine = products[group * most + pair - qo[group]]
    out.copy_(torch.where(valid, mine.to(out.dtype), out))
    return out


# ---------------------------------------------------------------- in 64 bits, from the definition
def exact(case, seed):
    state = prepare(case, seed)
    op, dim = state["op"], state["dim"]
    nb = blocks_of(dim)

    def two_to(e):
        return ((e.long() + 1023) << 52).view(torch.float64)

    def encode(x):
        """Nearest e4m3 values and the exponent of their scale, in float64."""
        x = x.double()
        x = torch.cat([x, x.new_zeros(len(x), nb * BLOCK - dim)], 1).view(len(x), nb, BLOCK)
        part, e = torch.frexp(x.abs().max(2).values / 448.0)
        e = torch.where(part == 0.5, e - 1, e)
        e = torch.where(part == 0.0, torch.full_like(e, -127), e).clamp_min(-127)
        y = x / two_to(e)[:, :, None]
        step = two_to((torch.frexp(y)[1] - 1).clamp_min(-6) - 3)  # e4m3: 3 bits below the first, down to 2^-9
        return torch.round(y / step) * step, e

    def decode(codes, scales):
        scale = two_to(scales[:, :nb].int() - 127)
        return (codes.to(torch.float32).double().view(len(codes), nb, BLOCK) * scale[:, :, None]).view(len(codes), -1)

    def both():
        if state["query_scales"] is not None:
            q = decode(state["queries"], state["query_scales"])
        else:
            y, e = encode(state["queries"])
            q = (y * two_to(e)[:, :, None]).view(len(y), -1)
        return q, decode(state["codes"], state["scales"])

    if op == "write":
        y, e = encode(state["rows"])
        codes = torch.zeros(state["codes"].shape, dtype=torch.float64, device=y.device)
        slots = state["slots"]
        slots = torch.arange(len(y), device=y.device) if slots is None else slots
        codes[slots[slots >= 0]] = y.view(len(y), -1)[slots >= 0]
        return {"codes": codes, "scales": None}
    if op == "read":
        slots = torch.arange(state["count"], device=state["codes"].device) if state["slots"] is None else state["slots"]
        codes = state["codes"].view(torch.uint8)[slots].view(torch.float8_e4m3fn)
        return decode(codes, state["scales"][slots])[:, :dim]
    q, r = both()
    if op == "scores":
        return q @ r.T
    qo, ro = offsets_of(case)
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device=q.device)
    for g in range(case["groups"]):
        if qo[g + 1] > qo[g] and ro[g + 1] > ro[g]:
            out[qo[g] : qo[g + 1], : ro[g + 1] - ro[g]] = q[qo[g] : qo[g + 1]] @ r[ro[g] : ro[g + 1]].T
    return out
