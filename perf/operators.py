"""The flat-scoring operators as they are measured: the cases, their inputs, a plain form of each and its 64-bit value.

Five operators over a table of records held as 8-bit codes with a scale each (`shine_amd.flat`):

* quantize  rows -> codes and scales: scale = f32(max|x| / 127), code = round-half-even(x / scale)
* score     the inner products of a query batch with every record, (float(sum qc*xc) * qscale) * xscale [+ bias]
* adjust    penalties for records a query has been shown, per-record biases, allowed-record bits
* topk      the k best of every row, ties to the lowest id; -inf and NaN are no answers (id -1, value -inf)
* search    score, adjust and topk in one call, from float queries

`own` False computes them with elementary torch operations, True with the framework's calls.
"""
import math
import sys

import torch

own = False
if "dm-hnsw-reference_amd" not in sys.path:
    sys.path.insert(1, "dm-hnsw-reference_amd")

NEG = float("-inf")


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a batch of queries in fp16, as the Text-to-Image configuration holds them, on their way to the product
        dict(name="quantize_batch", op="quantize", n=1024, dim=200, elem="float16"),
        # the table of the SIFT1M configuration, quantised once when it is opened
        dict(name="quantize_table", op="quantize", n=1_000_000, dim=128, elem="float32"),
        # one query against the siftsmall table: latency
        dict(name="score_one", op="score", nq=1, n=10_000, dim=128, elem="float32", out="float32", metric="ip"),
        # a batch of the SIFT1M configuration against a DEEP-shaped part of an odd size, L2 order through the bias
        dict(name="score_batch", op="score", nq=1024, n=100_003, dim=96, elem="float32", out="float32", metric="l2"),
        # long embeddings, 16-bit in and out: the product itself counts
        dict(name="score_wide", op="score", nq=2048, n=32_768, dim=1024, elem="bfloat16", out="bfloat16", metric="ip"),
        # one user's scores with everything on: latency
        dict(name="adjust_one", op="adjust", nq=1, n=50_000, elem="float32", seen=64, rows=True),
        # many users, long histories with repeats, a mask each, rows of an odd length
        dict(name="adjust_batch", op="adjust", nq=256, n=151_937, elem="bfloat16", seen=2048, rows=True),
        # one row of scores: latency
        dict(name="topk_one", op="topk", nq=1, n=100_000, k=10, elem="float32"),
        # a batch of rows, a long answer (the k = 100 of ground-truth files), rows of an odd length
        dict(name="topk_batch", op="topk", nq=1024, n=100_003, k=100, elem="float32"),
        # one query against the whole SIFT1M-shaped table: latency, the table's bytes count
        dict(name="search_one", op="search", nq=1, n=1_000_000, dim=128, k=10, elem="float32", metric="l2", seen=0,
             filter="none"),
        # the batch of the SIFT1M configuration with one filter for all
        dict(name="search_batch", op="search", nq=1024, n=1_000_000, dim=128, k=10, elem="float32", metric="l2", seen=0,
             filter="shared"),
        # Text-to-Image-shaped fp16 inner products with a mask, a bias and a history for each user
        dict(name="search_users", op="search", nq=256, n=200_000, dim=200, k=100, elem="float16", metric="ip", seen=256,
             filter="rows"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "score", "adjust", "topk", "search"])
    elem = rng.choice(["float32", "float16", "bfloat16"])
    if op == "quantize":
        dim = _log(rng, 8, 1100)
        return dict(op=op, n=min(_log(rng, 1, 1_000_000), 128_000_000 // dim), dim=dim, elem=elem)
    if op == "score":
        nq, dim = _log(rng, 1, 4096), _log(rng, 16, 1100)
        n = min(_log(rng, 1000, 1_000_000), 100_000_000 // nq)
        return dict(op=op, nq=nq, n=n, dim=dim, elem=elem, out=rng.choice(["float32", "float16", "bfloat16"]),
                    metric=rng.choice(["ip", "l2"]))
    if op == "adjust":
        nq = _log(rng, 1, 1024)
        return dict(op=op, nq=nq, n=min(_log(rng, 500, 500_000), 60_000_000 // nq), elem=elem,
                    seen=rng.choice([0, _log(rng, 1, 4096)]), rows=rng.random() < 0.5)
    if op == "topk":
        nq = _log(rng, 1, 4096)
        return dict(op=op, nq=nq, n=min(_log(rng, 200, 1_000_000), 100_000_000 // nq), k=_log(rng, 1, 256), elem=elem)
    nq, dim = _log(rng, 1, 2048), _log(rng, 16, 256)
    n = min(_log(rng, 1000, 1_000_000), 400_000_000 // nq)
    return dict(op=op, nq=nq, n=n, dim=dim, k=_log(rng, 1, 256), elem=elem, metric=rng.choice(["ip", "l2"]),
                seen=rng.choice([0, 0, _log(rng, 1, 512)]), filter=rng.choice(["none", "shared", "rows"]))


def work(case):
    c = case
    size = {"float32": 4, "float16": 2, "bfloat16": 2}
    if c["op"] == "quantize":
        return {"bytes": c["n"] * (c["dim"] * (size[c["elem"]] + 1) + 4), "flops": 2 * c["n"] * c["dim"]}
    if c["op"] == "score":
        return {"bytes": c["nq"] * c["dim"] * size[c["elem"]] + c["n"] * (c["dim"] + 4) +
                (4 * c["n"] if c["metric"] == "l2" else 0) + c["nq"] * c["n"] * size[c["out"]],
                "flops": 2 * c["nq"] * c["n"] * c["dim"]}
    if c["op"] == "adjust":
        masks = (c["nq"] if c["rows"] else 1) * ((c["n"] + 31) // 32) * 4
        return {"bytes": 2 * c["nq"] * c["n"] * size[c["elem"]] + masks + 4 * c["n"] + 4 * c["nq"] * c["seen"],
                "flops": 2 * c["nq"] * c["n"]}
    if c["op"] == "topk":
        return {"bytes": c["nq"] * c["n"] * size[c["elem"]] + c["nq"] * c["k"] * (size[c["elem"]] + 4),
                "flops": c["nq"] * c["n"]}
    masks = {"none": 0, "shared": 1, "rows": c["nq"]}[c["filter"]] * ((c["n"] + 31) // 32) * 4
    return {"bytes": c["nq"] * c["dim"] * size[c["elem"]] + c["n"] * (c["dim"] + 8) + masks + 4 * c["nq"] * c["seen"] +
            8 * c["nq"] * c["k"], "flops": 2 * c["nq"] * c["n"] * c["dim"]}


# ---------------------------------------------------------------- inputs

def _rows(g, n, dim, elem, centres):
    """Embedding-like rows: a mixture in a low-dimensional latent space with a decaying spectrum, unit norm."""
    latent = min(dim, 48)
    model = torch.Generator(device="cuda")
    model.manual_seed(77)
    c = torch.randn((512, latent), generator=model, device="cuda") * 2.5
    p = torch.randn((latent, dim), generator=model, device="cuda")
    spectrum = torch.arange(1, latent + 1, device="cuda", dtype=torch.float32) ** -0.5
    label = torch.randint(0, centres, (n,), generator=g, device="cuda")
    x = (c[label] + torch.randn((n, latent), generator=g, device="cuda")) * spectrum @ p
    return (x / x.norm(dim=1, keepdim=True).clamp_min(1e-12)).to(getattr(torch, elem))


def _bits(g, rows, n, share):
    """Packed allowed-record bits, int32 words, bit i % 32 of word i // 32 for record i."""
    words = (n + 31) // 32
    out = torch.zeros((rows, words), dtype=torch.int32, device="cuda")
    for b in range(32):
        on = torch.rand((rows, words), generator=g, device="cuda") < share
        out |= on.to(torch.int32) << b
    return out


def _history(g, nq, n, length):
    """Shown records: a skewed draw with repeats, the tail of every row padded with -1."""
    u = torch.rand((nq, length), generator=g, device="cuda")
    ids = (u * u * u * n).to(torch.int32).clamp_(0, n - 1)
    lengths = torch.randint(length // 2, length + 1, (nq, 1), generator=g, device="cuda")
    return torch.where(torch.arange(length, device="cuda") < lengths, ids, -1).to(torch.int32)


def _penalties(g, nq):
    return dict(repetition=1.0 + torch.rand(nq, generator=g, device="cuda"),
                frequency=0.05 * torch.rand(nq, generator=g, device="cuda"),
                presence=0.1 * torch.rand(nq, generator=g, device="cuda"))


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case=c)
    if c["op"] == "quantize":
        s["rows"] = _rows(g, c["n"], c["dim"], c["elem"], 512)
        return s
    if c["op"] in ("score", "search"):
        rows = _rows(g, c["n"], c["dim"], c["elem"], 512)
        s["queries"] = _rows(g, c["nq"], c["dim"], c["elem"], 512)
        if own:  # the table is laid out once, when it is opened
            from shine_amd import flat
            s["table"] = flat.FlatTable(rows, metric=c["metric"])
        else:
            s["codes"], s["scales"] = _quantize(rows)
            s["norms"] = _half_norms(s["codes"], s["scales"]) if c["metric"] == "l2" else None
    if c["op"] in ("adjust", "topk"):
        x = torch.randn((c["nq"], c["n"]), generator=g, device="cuda") * 0.3
        if c["op"] == "topk":  # a filter has been over the rows
            x = torch.where(torch.rand((c["nq"], 1), generator=g, device="cuda") < 0.5, x,
                            torch.where(x > -0.3, x, NEG))
        s["scores"] = x.to(getattr(torch, c["elem"]))
    if c["op"] == "adjust":
        s["adjust"] = dict(bias=torch.randn(c["n"], generator=g, device="cuda") * 0.1,
                           allow=_bits(g, c["nq"] if c["rows"] else 1, c["n"], 0.7))
        if c["seen"]:
            s["adjust"].update(seen=_history(g, c["nq"], c["n"], c["seen"]), **_penalties(g, c["nq"]))
    if c["op"] == "search":
        s["adjust"] = {}
        if c["filter"] != "none":
            s["adjust"]["allow"] = _bits(g, c["nq"] if c["filter"] == "rows" else 1, c["n"], 0.4)
        if c["filter"] == "rows":
            s["adjust"]["bias"] = torch.randn(c["n"], generator=g, device="cuda") * 0.02
        if c["seen"]:
            s["adjust"].update(seen=_history(g, c["nq"], c["n"], c["seen"]), **_penalties(g, c["nq"]))
    return s


# ---------------------------------------------------------------- plain forms

def _quantize(rows):
    """The borders between codes are met in 64 bits."""
    x = rows.double()
    scales = (x.abs().amax(1) / 127.0).float()
    codes = torch.round(x / scales.double().clamp_min(1e-300)[:, None]).clamp_(-127, 127)
    return codes.to(torch.int8), scales


def _half_norms(codes, scales):
    """-|x|^2 / 2 of the rows that the codes stand for: added to an inner product it gives the order of L2 distances."""
    squares = codes.float().square().sum(1) if codes.shape[1] <= 1040 else codes.double().square().sum(1).float()
    return -0.5 * (squares * scales * scales)


def _scores(codes, scales, norms, queries):
    qc, qs = _quantize(queries)
    wide = codes.shape[1] > 1040  # sums that pass 2^24
    acc = (qc.double() @ codes.double().T).float() if wide else qc.float() @ codes.float().T
    s = (acc * qs[:, None]) * scales
    return s if norms is None else s + norms


def _adjust(s, bias=None, allow=None, seen=None, repetition=None, frequency=None, presence=None):
    nq, n = s.shape
    if seen is not None:
        at = torch.where(seen >= 0, seen, n).long()
        counts = torch.zeros((nq, n + 1), device="cuda").scatter_add_(1, at, torch.ones(at.shape, device="cuda"))[:, :n]
        r = repetition[:, None]
        p = torch.where(s > 0, s / r, s * r) - frequency[:, None] * counts - presence[:, None]
        s = torch.where(counts > 0, p, s)
    if bias is not None:
        s = s + bias
    if allow is not None:
        i = torch.arange(n, device="cuda")
        s = torch.where(((allow[:, i >> 5] >> (i & 31)) & 1) != 0, s, NEG)
    return s


def _topk(s, k):
    """One 64-bit key for each entry: the value's order above, the id's inverse below, so that ties go to the lowest."""
    n = s.shape[1]
    s = torch.where(s.isnan(), NEG, s.float()) + 0.0
    b = s.view(torch.int32)
    order = b ^ ((b >> 31) & 0x7FFFFFFF)
    keys = (order.long() << 32) | (0x7FFFFFFF - torch.arange(n, device="cuda"))
    keys = torch.topk(keys, min(k, n), dim=1).values
    ids = (0x7FFFFFFF - (keys & 0xFFFFFFFF)).int()
    b = (keys >> 32).int()
    values = (b ^ ((b >> 31) & 0x7FFFFFFF)).view(torch.float32)
    ids = torch.where(values == NEG, -1, ids)
    return torch.nn.functional.pad(values, (0, max(0, k - n)), value=NEG), torch.nn.functional.pad(ids, (0, max(0, k - n)), value=-1)


def run(state):
    c = state["case"]
    if own:
        return _run_own(c, state)
    if c["op"] == "quantize":
        codes, scales = _quantize(state["rows"])
        return codes * scales[:, None]
    if c["op"] == "score":
        return _scores(state["codes"], state["scales"], state["norms"], state["queries"]).to(getattr(torch, c["out"]))
    if c["op"] == "adjust":
        return _adjust(state["scores"].float(), **state["adjust"]).to(getattr(torch, c["elem"]))
    if c["op"] == "topk":
        values, ids = _topk(state["scores"], c["k"])
        return values.to(getattr(torch, c["elem"])), ids
    s = _scores(state["codes"], state["scales"], state["norms"], state["queries"])
    return _topk(_adjust(s, **state["adjust"]), c["k"])


def _run_own(c, state):
    from shine_amd import flat
    if c["op"] == "quantize":
        codes, scales = flat.quantize_rows(state["rows"])
        return codes * scales[:, None]
    if c["op"] == "score":
        return flat.scores(state["table"], state["queries"], dtype=getattr(torch, c["out"]))
    if c["op"] == "adjust":
        return flat.adjust(state["scores"], **state["adjust"])
    if c["op"] == "topk":
        return flat.topk(state["scores"], c["k"])
    return flat.search(state["table"], state["queries"], c["k"], **state["adjust"])


# ---------------------------------------------------------------- the values in 64 bits

def _exact_codes(rows):
    """codes and scales as the definition has them: the scale is a 32-bit number, the quotient is not rounded first."""
    x = rows.to(torch.float64)
    scale = torch.div(torch.linalg.vector_norm(x, ord=math.inf, dim=1), 127.0).to(torch.float32).to(torch.float64)
    quotient = torch.where(scale[:, None] > 0, x / scale[:, None], torch.zeros_like(x))
    floor = torch.floor(quotient)
    part = quotient - floor
    up = (part > 0.5) | ((part == 0.5) & (torch.remainder(floor, 2) == 1))
    return (floor + up).clamp(-127, 127), scale


def exact(case, seed):
    global own
    c, was = case, own
    own = False
    s = prepare(case, seed)
    own = was
    if c["op"] == "quantize":
        codes, scale = _exact_codes(s["rows"])
        return codes * scale[:, None]
    if c["op"] == "topk":
        x = s["scores"].to(torch.float64)
        k = min(c["k"], c["n"])
        best = torch.sort(torch.topk(x, k, dim=1).values, dim=1, descending=True).values
        return torch.cat([best, torch.full((c["nq"], c["k"] - k), NEG, dtype=torch.float64, device="cuda")], 1), None
    if c["op"] == "adjust":
        x = s["scores"].to(torch.float64)
    else:
        qc, qs = _exact_codes(s["queries"])
        xc, xs = s["codes"].to(torch.float64), s["scales"].to(torch.float64)
        q, x = qc * qs[:, None], xc * xs[:, None]
        x, half = q @ x.T.contiguous(), x.square().sum(1) / 2
        if c["metric"] == "l2":
            x -= half
        if c["op"] == "score":
            return x
    a = s["adjust"]
    if "seen" in a:
        # the records a row has been shown, sorted: a run of equal ids is one record and its length the count
        ids, _ = a["seen"].to(torch.int64).sort(dim=1)
        for row in range(c["nq"]):
            who, times = torch.unique_consecutive(ids[row][ids[row] >= 0], return_counts=True)
            old, r = x[row, who], a["repetition"][row].double()
            new = torch.where(old > 0, old / r, old * r)
            x[row, who] = new - times.double() * a["frequency"][row].double() - a["presence"][row].double()
    if "bias" in a:
        x += a["bias"].to(torch.float64)
    if "allow" in a:
        shifts = torch.arange(32, device="cuda", dtype=torch.int32)
        for row in range(0, c["nq"], 64):
            words = a["allow"][row:row + 64] if a["allow"].shape[0] > 1 else a["allow"]
            on = (words[:, :, None].bitwise_right_shift(shifts) & 1).flatten(1)[:, :c["n"]].bool()
            x[row:row + 64].masked_fill_(~on, NEG)
    if c["op"] == "adjust":
        return x
    k = min(c["k"], c["n"])
    best = torch.topk(x, k, dim=1).values.sort(dim=1, descending=True).values
    # which of two records nearer than 32 bits comes first is no number
    return torch.cat([best, torch.full((c["nq"], c["k"] - k), NEG, dtype=torch.float64, device="cuda")], 1), None
