"""Flat scoring on the GPU against a plain implementation in 64 bits.

Tolerances: a rounding to a type is off by at most u = finfo(type).eps / 2 of the value.  f32 steps: u32 = 2^-24.
* quantisation: the codes are defined in real arithmetic on 32-bit numbers: they have to be equal.
* scores: the sum of products is exact; its conversion, two products and (L2) one sum are rounded to f32:
  3 u32 |p| (1 + 3 u32) for the product p, u32 |v| for the sum, then u |v| for the output type.
* adjust: at most 6 f32 roundings, of values no larger than M = |s'| + |f c| + |p| + |b|; then u |v|.
* top-k and search: values and ids equal those of the scores that they rank.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

NEG = -math.inf
U32 = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def F():
    from shine_amd import flat
    return flat


def rows(n, dim, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((n, dim), generator=g) * scale).to(dtype)


# ---- the plain forms, in 64 bits on the CPU

def codes64(x):
    """codes (float64) and scales (float64 holding f32 numbers)"""
    x = x.double()
    scale = (x.abs().amax(1) / 127).float().double()
    q = x / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    return torch.where(scale[:, None] > 0, torch.round(q).clamp(-127, 127), torch.zeros_like(q)), scale


def scores64(table, q, metric):
    """exact scores, and the largest error that f32 steps may bring"""
    xc, xs = codes64(table)
    qc, qs = codes64(q)
    p = (qc @ xc.T) * qs[:, None] * xs[None, :]
    err = 3 * U32 * p.abs() * (1 + 3 * U32)
    if metric == "l2":
        half = xc.square().sum(1) * xs * xs / 2
        p = p - half
        err = err + 3 * U32 * half * (1 + 3 * U32) + U32 * (p.abs() + err)  # the half norm: a conversion, two products
    return p, err


def scores32(table, q, metric):
    """the same in f32, step by step as the definition rounds"""
    xc, xs = codes64(table)
    qc, qs = codes64(q)
    s = ((qc @ xc.T).float() * qs.float()[:, None]) * xs.float()[None, :]
    if metric == "l2":
        s = s + (-0.5 * ((xc.square().sum(1).float() * xs.float()) * xs.float()))
    return s


def adjust64(s, bias=None, allow=None, seen=None, repetition=None, frequency=None, presence=None):
    s = s.double().clone()
    nq, n = s.shape
    big = torch.zeros_like(s)
    for i in range(nq):
        if seen is not None:
            ids, c = np.unique([x for x in seen[i % seen.shape[0]].tolist() if 0 <= x < n], return_counts=True)
            for j, m in zip(ids.astype(int), c):
                r = float(repetition[i]) if repetition is not None else 1.0
                f = float(frequency[i]) if frequency is not None else 0.0
                p = float(presence[i]) if presence is not None else 0.0
                v = s[i, j].item()
                v = v / r if v > 0 else v * r
                s[i, j] = v - f * m - p
                big[i, j] = abs(f * m) + abs(p) + abs(v)
    big = torch.maximum(big, s.abs())
    if bias is not None:
        b = bias.double().reshape(-1, n)
        s = s + b
        big = big + b.abs()
    if allow is not None:
        a = allow.reshape(-1, allow.shape[-1]).numpy().view(np.uint32)
        on = np.unpackbits(a.view(np.uint8), axis=1, bitorder="little")[:, :n].astype(bool)
        s = torch.where(torch.from_numpy(on).expand(nq, n), s, torch.tensor(NEG, dtype=torch.float64))
    return s, 6 * U32 * big


def topk_plain(s, k):
    """by (value descending, id ascending); -inf and NaN are no answers"""
    s = s.float().numpy() + np.float32(0)
    nq, n = s.shape
    values = np.full((nq, k), -np.inf, np.float32)
    ids = np.full((nq, k), -1, np.int32)
    for i in range(nq):
        ok = np.nonzero(s[i] > -np.inf)[0]
        order = ok[np.lexsort((ok, -s[i][ok].astype(np.float64)))][:k]
        values[i, :len(order)] = s[i][order]
        ids[i, :len(order)] = order
    return torch.from_numpy(values), torch.from_numpy(ids)


def close(got, want, err, dtype):
    got, want = got.double().cpu(), want
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * u  # half a step below the normal numbers
    same = (got == want) | (got.isnan() & want.isnan())
    off = (got - want).abs()
    bound = err * (1 + u) + u * want.abs() + tiny
    bad = ~same & ~(off <= bound)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], bound[bad][:4])


def bits(n, nq, share, seed):
    g = np.random.default_rng(seed)
    on = g.random((nq, n)) < share
    packed = np.packbits(np.pad(on, ((0, 0), (0, (-n) % 32))), axis=1, bitorder="little")
    return torch.from_numpy(packed.copy().view(np.int32)), on


# ---- quantisation

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (3, 7), (1, 64), (5, 65), (33, 96), (17, 100), (130, 128), (65, 200), (9, 256),
                                   (4, 257), (3, 1000), (2, 1025), (2, 16384)])
def test_quantize_equals_the_definition(n, dim, dtype):
    x = rows(n, dim, n * 1000 + dim, dtype)
    codes, scales = F().quantize_rows(x.cuda())
    want, scale = codes64(x)
    assert codes.shape == (n, dim) and scales.shape == (n,)
    assert torch.equal(codes.cpu().double(), want)
    assert torch.equal(scales.cpu().double(), scale)


def test_quantize_halves_go_to_even_and_borders_are_exact():
    """Rows with 127 as their largest have scale 1: halves are exact ties.  A second row is built next to its borders."""
    halves = torch.arange(-126.5, 127, 1.0)
    x = torch.stack([torch.cat([torch.tensor([127.0]), halves, torch.zeros(1)])] * 2)
    s = torch.tensor(0.37, dtype=torch.float32)
    edge = (halves.double() * s.double()).float()
    near = torch.cat([torch.tensor([127.0]) * s, edge, torch.zeros(1)])
    up, down = torch.nextafter(near, torch.full_like(near, 1e9)), torch.nextafter(near, torch.full_like(near, -1e9))
    up[0] = down[0] = near[0]
    x = torch.cat([x, torch.stack([near, up, down])])
    codes, scales = F().quantize_rows(x.cuda())
    want, scale = codes64(x)
    assert torch.equal(scales.cpu().double(), scale)
    assert torch.equal(codes.cpu().double(), want)


def test_quantize_extreme_rows():
    big, tiny = torch.finfo(torch.float32).max, 2.0 ** -149
    x = torch.tensor([[0.0, -0.0, 0.0], [big, -big, big / 3], [tiny, 0.0, -tiny], [tiny * 100, tiny * 200, -tiny * 50],
                      [1e-35, -3e-36, 2e-36], [1e-29, 3e-31, -7e-30], [1.0, math.nan, 0.0], [math.inf, 1.0, 2.0],
                      [-math.inf, math.nan, 1.0]])
    codes, scales = F().quantize_rows(x.cuda())
    want, scale = codes64(x[:6])
    assert torch.equal(scales[:6].cpu().double(), scale)
    assert torch.equal(codes[:6].cpu().double(), want)
    assert scales[6:].isnan().all() and not codes[6:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strided_rows(dtype):
    """rows at every address that the type allows, with a stride of their own"""
    base = rows(20, 150, 5, dtype)
    for off, dim in ((0, 100), (1, 96), (3, 128), (7, 65)):
        x = base[:, off:off + dim]
        codes, scales = F().quantize_rows(base.cuda()[:, off:off + dim])
        want, scale = codes64(x)
        assert torch.equal(codes.cpu().double(), want) and torch.equal(scales.cpu().double(), scale)


# ---- scores

SCORE_SIZES = [(1, 1, 1), (1, 33, 8), (2, 31, 64), (1, 1000, 128), (5, 130, 96), (16, 257, 100), (17, 300, 200), (63, 65, 65),
               (64, 128, 256), (65, 129, 300), (130, 515, 128), (3, 2000, 1024), (70, 140, 1025), (2, 40, 4096),
               (200, 33, 513), (257, 1030, 96)]


@pytest.mark.parametrize("metric", ["ip", "l2"])
@pytest.mark.parametrize("nq,n,dim", SCORE_SIZES)
def test_scores(nq, n, dim, metric):
    x, q = rows(n, dim, dim + n), rows(nq, dim, dim + nq + 7)
    table = F().FlatTable(x.cuda(), metric=metric)
    want, err = scores64(x, q, metric)
    s = F().scores(table, q.cuda())
    close(s, want, err, torch.float32)
    assert torch.equal(s.cpu(), scores32(x, q, metric))
    for dtype in (torch.float16, torch.bfloat16):
        t = F().scores(table, q.cuda(), dtype=dtype)
        close(t, want, err, dtype)
        assert torch.equal(t, s.to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_of_each_query_type(dtype):
    x, q = rows(150, 200, 1, dtype), rows(40, 200, 2, dtype)
    table = F().FlatTable(x.cuda())
    assert torch.equal(F().scores(table, q.cuda()).cpu(), scores32(x, q, "ip"))


def test_scores_largest_sums():
    """every product at its largest: the sums pass 2^24 and stay exact"""
    for dim in (1040, 1041, 16384):
        x = torch.ones(3, dim)
        x[1] = -1
        table = F().FlatTable(x.cuda())
        want, err = scores64(x, x, "ip")
        s = F().scores(table, x.cuda())
        close(s, want, err, torch.float32)
        assert torch.equal(s.cpu(), scores32(x, x, "ip"))


def test_scores_of_rows_without_a_scale():
    x = rows(10, 32, 3)
    x[2] = 0
    x[5, 7] = math.nan
    q = rows(4, 32, 4)
    q[1] = 0
    q[3, 0] = math.inf
    s = F().scores(F().FlatTable(x.cuda(), metric="l2"), q.cuda()).cpu()
    assert s[3].isnan().all() and s[:, 5].isnan().all()
    keep = [0, 1, 2, 3, 4, 6, 7, 8, 9]
    assert torch.equal(s[:3][:, keep], scores32(x[keep], q[:3], "l2"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,n,dim", [(3, 45, 96), (70, 301, 128), (20, 64, 300)])
def test_scores_into_a_strided_out(dtype, nq, n, dim):
    """rows of an odd stride at an odd place: nothing beside them is written"""
    x, q = rows(n, dim, 8), rows(nq, dim, 9)
    table = F().FlatTable(x.cuda())
    whole = torch.full((nq + 2, n + 13), 7.0, dtype=dtype, device="cuda")
    out = whole[1:nq + 1, 5:5 + n]
    assert F().scores(table, q.cuda(), out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out, F().scores(table, q.cuda(), dtype=dtype))
    whole[1:nq + 1, 5:5 + n] = 7.0
    assert (whole == 7.0).all()


# ---- adjust

def adjustments(nq, n, seed, h=0, bias=None, allow=None):
    g = torch.Generator().manual_seed(seed)
    a = {}
    if bias:
        a["bias"] = torch.randn((n,) if bias == "shared" else (nq, n), generator=g) * 0.2
    if allow:
        a["allow"] = bits(n, 1 if allow == "shared" else nq, 0.6, seed)[0]
    if h:
        a["seen"] = torch.randint(-2, min(n, 2 * h) + 3, (nq, h), generator=g, dtype=torch.int32)
        a["repetition"] = 1 + torch.rand(nq, generator=g)
        a["frequency"] = torch.rand(nq, generator=g) * 0.1
        a["presence"] = torch.rand(nq, generator=g) * 0.2
    return a


def cuda(a):
    return {k: v.cuda() for k, v in a.items()}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,n", [(1, 1), (1, 31), (2, 33), (3, 4095), (1, 4097), (5, 8191), (2, 20003)])
@pytest.mark.parametrize("h,bias,allow", [(0, "shared", None), (0, None, "rows"), (1, None, None), (40, "rows", "shared"),
                                          (700, "shared", "rows")])
def test_adjust(dtype, nq, n, h, bias, allow):
    s = rows(nq, n, nq + n, dtype)
    a = adjustments(nq, n, n + h, h, bias, allow)
    want, err = adjust64(s, **a)
    close(F().adjust(s.cuda(), **cuda(a)), want, err, dtype)


def test_adjust_one_at_a_time_and_in_place():
    s = rows(4, 5000, 1)
    a = adjustments(4, 5000, 2, 30, "rows", "rows")
    for some in ([], ["seen"], ["seen", "repetition"], ["seen", "frequency"], ["seen", "presence"], ["bias"], ["allow"]):
        b = {k: a[k] for k in some}
        want, err = adjust64(s, **b)
        close(F().adjust(s.cuda(), **cuda(b)), want, err, torch.float32)
    x = s.cuda()
    want = F().adjust(x, **cuda(a))
    assert F().adjust(x, **cuda(a), out=x) is x
    assert torch.equal(x, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_adjust_special_values(dtype):
    """masks win over everything, infinities and NaN pass, the type's lowest value stays, counts of one id in thousands"""
    n = 300
    s = rows(3, n, 4, dtype)
    s[0, 0], s[0, 1], s[0, 2], s[0, 3] = math.nan, math.inf, NEG, torch.finfo(dtype).min
    s[1, :4] = s[0, :4]
    s[1, 4] = 0.0
    allow, on = bits(n, 3, 0.5, 6)
    a = allow.numpy().view(np.uint32)
    a[0, 0] &= ~np.uint32(0xF)   # row 0: the special values are masked
    a[1, 0] |= np.uint32(0xFF)   # row 1: they are not
    a[2] = 0                     # row 2: nothing is left
    seen = torch.full((3, 5000), 4, dtype=torch.int32)
    arg = dict(allow=allow, seen=seen, repetition=torch.full((3,), 2.0), frequency=torch.full((3,), 0.25),
               presence=torch.full((3,), 0.5))
    got = F().adjust(s.cuda(), **cuda(arg))
    want, err = adjust64(s, **arg)
    close(got, want, err, dtype)
    assert (got[2] == NEG).all() and (got[0, :4] == NEG).all()
    assert got[1, 0].isnan() and got[1, 1] == math.inf and got[1, 2] == NEG and got[1, 3] == torch.finfo(dtype).min
    values, ids = F().topk(got, 5)
    assert (ids[2] == -1).all() and (values[2] == NEG).all()


def test_adjust_longest_history():
    """65,535 ids of one record, beside one that shares its count's word and one met once"""
    s = rows(2, 9000, 4)
    seen = torch.full((2, 65535), 4098, dtype=torch.int32)
    seen[1, :30000] = 4099
    seen[1, 7] = 8999
    arg = dict(seen=seen, frequency=torch.tensor([1e-3, 1.0]))
    want, err = adjust64(s, **arg)
    close(F().adjust(s.cuda(), **cuda(arg)), want, err, torch.float32)
    table = F().FlatTable(rows(9000, 16, 1).cuda())
    q = rows(2, 16, 2).cuda()
    values, ids = F().search(table, q, 20, **cuda(arg))
    v, i = F().topk(F().adjust(F().scores(table, q), **cuda(arg)), 20)
    assert torch.equal(ids, i) and torch.equal(values, v)


def test_adjust_strides():
    whole = rows(7, 999, 3).cuda()
    s = whole[1:5, 3:903]
    a = adjustments(4, 900, 2, 30, "rows", "rows")
    big = {k: torch.zeros((v.shape[0], v.shape[1] + 9), dtype=v.dtype, device="cuda") for k, v in a.items() if v.dim() == 2}
    b = cuda(a)
    for k, v in big.items():
        v[:, 2:2 + a[k].shape[1]] = b[k]
        b[k] = v[:, 2:2 + a[k].shape[1]]
    out = torch.full((4, 1001), 5.0, device="cuda")
    F().adjust(s, **b, out=out[:, 1:901])
    assert torch.equal(out[:, 1:901], F().adjust(s.contiguous(), **cuda(a)))
    assert (out[:, 0] == 5).all() and (out[:, 901:] == 5).all()


# ---- top-k

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,n,k", [(1, 1, 1), (1, 1, 256), (2, 5, 3), (3, 64, 64), (1, 255, 256), (1, 256, 256), (1, 257, 256),
                                    (4, 1000, 10), (2, 4096, 100), (1, 4097, 1), (1, 70001, 256), (3, 30011, 17),
                                    (1100, 700, 9)])
def test_topk(dtype, nq, n, k):
    s = rows(nq, n, nq * 7 + n + k, dtype)  # 16-bit types: many ties
    values, ids = F().topk(s.cuda(), k)
    want_v, want_i = topk_plain(s, k)
    assert torch.equal(ids.cpu(), want_i)
    assert torch.equal(values.cpu().float(), want_v)
    assert values.dtype == dtype


@pytest.mark.parametrize("k", [1, 10, 100, 256])
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "two values", "few left", "none left", "specials"])
def test_topk_orders(order, k):
    n = 50001
    s = torch.arange(n, dtype=torch.float32) / 8 - 3000
    if order == "falling":
        s = s.flip(0)
    elif order == "equal":
        s = torch.full((n,), -1.5)
    elif order == "two values":
        s = torch.where(torch.arange(n) % 3 == 0, 1.0, -2.0)
    elif order == "few left":
        s = torch.where(torch.arange(n) % 9001 == 77, s, NEG)
    elif order == "none left":
        s = torch.full((n,), NEG)
    elif order == "specials":
        s[::7], s[1::11], s[2::5], s[3::13], s[4::17] = math.nan, NEG, 0.0, -0.0, -math.nan
        s[40000], s[100] = math.inf, math.inf
        s[5], s[6] = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
        s[s > 0] = torch.where(torch.arange(int((s > 0).sum())) < 150, s[s > 0], NEG)
    s = torch.stack([s, s.roll(333)])
    values, ids = F().topk(s.cuda(), k)
    want_v, want_i = topk_plain(s, k)
    assert torch.equal(ids.cpu(), want_i)
    assert torch.equal(values.cpu(), want_v)


def test_topk_of_strided_rows_and_no_columns():
    whole = rows(5, 3001, 3).cuda()
    s = whole[1:4, 7:2900]
    assert all(torch.equal(a, b) for a, b in zip(F().topk(s, 20), F().topk(s.contiguous(), 20)))
    values, ids = F().topk(whole[:, :0], 3)
    assert (ids == -1).all() and (values == NEG).all()
    assert F().topk(whole[:0], 3)[0].shape == (0, 3)


# ---- search: a run of all of them together

SEARCH = [(1, 1, 4, 1), (1, 100, 16, 10), (1, 40000, 128, 10), (3, 777, 96, 100), (17, 5000, 200, 256), (64, 4099, 128, 10),
          (65, 8300, 64, 37), (100, 2500, 300, 10), (2100, 600, 32, 5), (5, 3000, 1100, 20)]


@pytest.mark.parametrize("metric", ["ip", "l2"])
@pytest.mark.parametrize("nq,n,dim,k", SEARCH)
def test_search(nq, n, dim, k, metric):
    x, q = rows(n, dim, 2 * n + dim), rows(nq, dim, dim + 1)
    table = F().FlatTable(x.cuda(), metric=metric)
    values, ids = F().search(table, q.cuda(), k)
    want_v, want_i = topk_plain(scores32(x, q, metric), k)
    assert torch.equal(ids.cpu(), want_i)
    assert torch.equal(values.cpu(), want_v)
    if metric == "l2":  # the distances of the rows that the codes stand for, in 64 bits
        xc, xs = codes64(x)
        qc, qs = codes64(q)
        xd, qd = xc * xs[:, None], qc * qs[:, None]
        d = F().FlatTable.distances(table, values, qd.float().cuda()).cpu().double()
        m = min(k, n)
        want = (qd[:, None] - xd[want_i[:, :m].long()]).square().sum(2) if nq * m * dim < 1e8 else None
        if want is not None:
            size = qd.square().sum(1)[:, None] + 2 * qd.norm(dim=1)[:, None] * xd.norm(dim=1).max() + xd.square().sum(1).max()
            assert ((d[:, :m] - want).abs() <= (dim + 8) * 2 * U32 * size).all()


@pytest.mark.parametrize("nq,n,dim,k,h,bias,allow", [
    (1, 3000, 128, 10, 0, None, "shared"), (1, 50000, 96, 100, 20, "shared", "rows"), (40, 6000, 200, 50, 300, "shared", "rows"),
    (70, 5003, 64, 10, 0, "rows", "shared"), (33, 4097, 100, 256, 5, None, None), (130, 900, 128, 10, 64, "rows", "rows"),
    (9, 9000, 700, 12, 33, "shared", "shared")])
def test_search_with_adjustments(nq, n, dim, k, h, bias, allow):
    x, q = rows(n, dim, n), rows(nq, dim, nq)
    a = adjustments(nq, n, 3, h, bias, allow)
    flat = F()
    for metric in ("ip", "l2"):
        table = flat.FlatTable(x.cuda(), metric=metric)
        values, ids = flat.search(table, q.cuda(), k, **cuda(a))
        v, i = flat.topk(flat.adjust(flat.scores(table, q.cuda()), **cuda(a)), k)
        assert torch.equal(ids, i) and torch.equal(values, v)
        want, err = adjust64(scores32(x, q, metric), **a)
        live = ids.cpu() >= 0
        at = torch.where(live, ids.cpu(), 0).long()
        close(torch.where(live, values.cpu(), 0.0), torch.where(live, want.gather(1, at), 0.0), err.gather(1, at), torch.float32)


def test_search_rows_that_a_filter_leaves_empty_and_short():
    flat = F()
    n = 10000
    table = flat.FlatTable(rows(n, 96, 1).cuda())
    allow = torch.zeros((3, (n + 31) // 32), dtype=torch.int32)
    allow[1, 100], allow[1, 312] = 5, 1 << 15      # records 3200, 3202, 9999
    allow[2] = -1
    values, ids = flat.search(table, rows(3, 96, 2).cuda(), 10, allow=allow.cuda())
    assert (ids[0] == -1).all() and (values[0] == NEG).all()
    assert sorted(ids[1, :3].tolist()) == [3200, 3202, 9999] and (ids[1, 3:] == -1).all()
    assert (ids[2] >= 0).all()


def test_search_equal_records_come_in_id_order():
    x = rows(50, 64, 1).repeat(200, 1)  # every record 200 times
    table = F().FlatTable(x.cuda(), metric="l2")
    q = rows(20, 64, 2)
    values, ids = F().search(table, q.cuda(), 250)
    want_v, want_i = topk_plain(scores32(x, q, "l2"), 250)
    assert torch.equal(ids.cpu(), want_i) and torch.equal(values.cpu(), want_v)


def test_search_of_sorted_records():
    """every record better than all before it: the worst order for what is kept"""
    n = 30000
    x = torch.zeros(n, 16)
    x[:, 0] = torch.linspace(1, 2, n)
    q = torch.zeros(70, 16)
    q[:, 0] = 1
    q[1::2, 0] = -1
    for k in (10, 256):
        values, ids = F().search(F().FlatTable(x.cuda()), q.cuda(), k)
        want_v, want_i = topk_plain(scores32(x, q, "ip"), k)
        assert torch.equal(ids.cpu(), want_i) and torch.equal(values.cpu(), want_v)


@pytest.mark.parametrize("k", [1, 10, 256])
@pytest.mark.parametrize("n,every", [(30000, 8), (30000, 4), (270000, 9)])
def test_search_when_a_sample_misses_the_best(n, every, k):
    """Every `every`-th block of 32 records is poor: a threshold taken there lets nearly all others through."""
    x = rows(n, 32, 5) * 0.1
    x[:, 0] = torch.where((torch.arange(n) // 32) % every == 0, -1.0, 1.0)
    q = rows(33, 32, 6) * 0.1
    q[:, 0] = 1
    q[1] = -q[1]
    a = adjustments(33, n, 3, 40, "shared", "rows")
    flat = F()
    table = flat.FlatTable(x.cuda())
    values, ids = flat.search(table, q.cuda(), k)
    want_v, want_i = topk_plain(scores32(x, q, "ip"), k)
    assert torch.equal(ids.cpu(), want_i) and torch.equal(values.cpu(), want_v)
    values, ids = flat.search(table, q.cuda(), k, **cuda(a))
    v, i = flat.topk(flat.adjust(flat.scores(table, q.cuda()), **cuda(a)), k)
    assert torch.equal(ids, i) and torch.equal(values, v)


@pytest.mark.parametrize("n", [8193, 131072, 400001])
def test_search_of_many_records(n):
    """more passes, a mask that leaves some rows few records and one row none"""
    x, q = rows(n, 48, 7), rows(40, 48, 8)
    a = adjustments(40, n, 3, 100, "shared", "rows")
    a["allow"][3] = 0
    a["allow"][4, 1:] = 0
    a["allow"][5, 50:-50] = 0
    flat = F()
    for metric in ("ip", "l2"):
        table = flat.FlatTable(x.cuda(), metric=metric)
        s = flat.scores(table, q.cuda())
        assert torch.equal(s.cpu(), scores32(x, q, metric))
        for k in (1, 64, 65, 200):
            for some in ([], ["allow"], ["allow", "bias"], list(a)):
                b = {key: a[key].cuda() for key in some}
                values, ids = flat.search(table, q.cuda(), k, **b)
                v, i = flat.topk(flat.adjust(s, **b), k)
                assert torch.equal(ids, i) and torch.equal(values, v)


def test_search_with_scales_far_apart():
    """products that overflow or vanish in one order of multiplication: the answers are those of the scores"""
    x, q = rows(9000, 32, 7), rows(40, 32, 8)
    x *= 10.0 ** torch.linspace(-30, 30, 9000)[torch.randperm(9000, generator=torch.Generator().manual_seed(1))][:, None]
    q *= 10.0 ** torch.linspace(-37, 37, 40)[:, None]
    x[5], q[7] = 0, 0
    flat = F()
    for metric in ("ip", "l2"):
        table = flat.FlatTable(x.cuda(), metric=metric)
        s = flat.scores(table, q.cuda())
        for k in (10, 200):
            values, ids = flat.search(table, q.cuda(), k)
            v, i = flat.topk(s, k)
            assert torch.equal(ids, i) and torch.equal(values, v)


def test_search_with_records_and_queries_without_a_scale():
    for nq, n in ((4, 500), (40, 500), (40, 20000)):
        x, q = rows(n, 32, 3), rows(nq, 32, 4)
        x[7, 3], x[450, 0] = math.nan, math.inf
        q[2, 1] = math.nan
        values, ids = F().search(F().FlatTable(x.cuda()), q.cuda(), 256)
        rest = [i for i in range(nq) if i != 2]
        assert (ids[2] == -1).all()
        assert not ((ids == 7) | (ids == 450)).any() and (ids[rest] >= 0).all() and values[rest].isfinite().all()


def test_empty_tables_and_batches():
    flat = F()
    table = flat.FlatTable(torch.empty((0, 32), device="cuda"))
    q = rows(3, 32, 1).cuda()
    assert flat.scores(table, q).shape == (3, 0)
    values, ids = flat.search(table, q, 4)
    assert (ids == -1).all() and (values == NEG).all()
    table = flat.FlatTable(rows(10, 32, 1).cuda())
    assert flat.scores(table, q[:0]).shape == (0, 10)
    assert flat.search(table, q[:0], 4)[1].shape == (0, 4)


# ---- streams, graphs, refusals

def test_calls_on_other_streams_at_once():
    flat = F()
    table = flat.FlatTable(rows(40000, 128, 1).cuda(), metric="l2")
    qs = [rows(32, 128, 10 + i).cuda() for i in range(4)]
    want = [flat.search(table, q, 10) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = []
    for q, st in zip(qs, streams):
        with torch.cuda.stream(st):
            got.append([flat.search(table, q, 10) for _ in range(3)])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for values, ids in g:
            assert torch.equal(values, w[0]) and torch.equal(ids, w[1])


def test_captured_and_replayed():
    """two graphs with workspaces of their own, replayed with new inputs between the program's own calls"""
    flat = F()
    table = flat.FlatTable(rows(30000, 96, 1).cuda())
    a = cuda(adjustments(24, 30000, 5, 50, "shared", "rows"))
    buffers, graphs, outs = [], [], []
    for i in range(2):
        q = rows(24, 96, 20 + i).cuda()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            flat.topk(flat.adjust(flat.scores(table, q), **a), 10), flat.search(table, q, 10, **a)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s = flat.scores(table, q)
            outs.append((flat.topk(flat.adjust(s, **a), 10), flat.search(table, q, 10, **a)))
        buffers.append(q)
        graphs.append(g)
    for turn in range(4):
        for i in (0, 1):
            buffers[i].copy_(rows(24, 96, 100 + 10 * turn + i))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            values, ids = flat.search(table, buffers[i], 10, **a)
            for v, j in outs[i]:
                assert torch.equal(v, values) and torch.equal(j, ids)


def test_python_refusals():
    flat = F()
    x = rows(20, 32, 1).cuda()
    table = flat.FlatTable(x)
    with pytest.raises(ValueError, match="dim 31"):
        flat.scores(table, x[:, :31])
    with pytest.raises(ValueError, match="unit stride"):
        flat.quantize_rows(x.T)
    with pytest.raises(ValueError, match="gradient"):
        flat.scores(table, x.clone().requires_grad_())
    with pytest.raises(ValueError, match="k must"):
        flat.topk(x, 257)
    with pytest.raises(ValueError, match="k must"):
        flat.search(table, x, 0)
    with pytest.raises(ValueError, match="out must"):
        flat.scores(table, x, out=torch.empty(20, 21, device="cuda"))
    with pytest.raises(ValueError, match="allow"):
        flat.adjust(x, allow=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="bias"):
        flat.adjust(x, bias=torch.zeros(32, dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError, match="bias"):
        flat.adjust(x, bias=torch.zeros(32))
    with pytest.raises(ValueError, match="needs seen"):
        flat.adjust(x, presence=torch.zeros(20, device="cuda"))
    with pytest.raises(ValueError, match="repetition"):
        flat.adjust(x, seen=torch.zeros((20, 1), dtype=torch.int32, device="cuda"), repetition=torch.ones(19, device="cuda"))
    with pytest.raises(Exception, match="stride"):
        flat.topk(x[:1].expand(5, 32), 3)


# More than 32 queries: lines of 128 bytes, whole ones and the rows' ends; runs of one line and of many.
LINES = [(33, 1, 64), (33, 31, 64), (64, 32, 128), (65, 33, 96), (33, 63, 128), (40, 64, 64), (100, 129, 100), (70, 1000, 128),
         (64, 4099, 30), (33, 700, 150), (50, 999, 256), (2000, 17003, 16), (1990, 17001, 200)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,n,dim", LINES)
def test_scores_in_rows_that_start_anywhere(dtype, nq, n, dim):
    x, q = rows(n, dim, n + dim), rows(nq, dim, nq)
    want = scores32(x, q, "l2").to(dtype)  # each step rounds as the definition does: equal bits
    t = F().FlatTable(x.cuda(), metric="l2")
    for before, ld in ((0, n), (1, n + 1), (2, n + 5), (7, n + 16)):
        room = torch.full((before + nq * ld + 3,), 7.0, dtype=dtype, device="cuda")
        out = room[before:before + nq * ld].view(nq, ld)[:, :n]
        F().scores(t, q.cuda(), out=out)
        got = room.cpu()
        assert torch.equal(got[before:before + nq * ld].view(nq, ld)[:, :n], want), (before, ld)
        assert bool((got[:before] == 7).all()) and bool((got[before + nq * ld:] == 7).all())
        assert bool((got[before:before + nq * ld].view(nq, ld)[:, n:] == 7).all()), "written behind a row"


# Searches of several passes, bit for bit as step by step: every width of rows, masks of each kind, parts of a block.
@pytest.mark.parametrize("dim", [40, 128, 150, 256])
@pytest.mark.parametrize("nq,n,k,h,bias,allow", [
    (20, 9001, 1, 0, None, "rows"), (40, 20017, 100, 30, "shared", "rows"), (130, 70003, 10, 300, None, "shared"),
    (300, 33000, 256, 5, "shared", "rows"), (65, 300001, 17, 0, None, None), (33, 8200, 3, 4096, None, None),
    (17, 12345, 40, 4097, None, "shared")])
def test_search_of_several_passes_with_adjustments(dim, nq, n, k, h, bias, allow):
    flat = F()
    table = flat.FlatTable(rows(n, dim, n + 1).cuda(), metric="l2")
    q = rows(nq, dim, nq + 2).cuda()
    a = cuda(adjustments(nq, n, 4, h, bias, allow))
    values, ids = flat.search(table, q, k, **a)
    s = flat.scores(table, q)
    v, i = flat.topk(flat.adjust(s, **a) if a else s, k)
    assert torch.equal(ids, i) and torch.equal(values, v)


@pytest.mark.parametrize("dim", [64, 200])
def test_search_of_several_passes_with_little_left(dim):
    flat = F()
    n, k = 40011, 8
    table = flat.FlatTable(rows(n, dim, 1).cuda())
    left = [[], [40010], [0, 31, 32, 20000, 40000, 40009, 40010], list(range(17, n, 1500)), list(range(39000, n))]
    allow = torch.zeros((20, (n + 31) // 32), dtype=torch.int64)
    for i in range(20):
        for j in left[i % 5]:
            allow[i, j // 32] |= 1 << (j % 32)
    allow = torch.where(allow >= 2 ** 31, allow - 2 ** 32, allow).int().cuda()
    q = rows(20, dim, 2).cuda()
    values, ids = flat.search(table, q, k, allow=allow)
    v, i = flat.topk(flat.adjust(flat.scores(table, q), allow=allow), k)
    assert torch.equal(ids, i) and torch.equal(values, v)
    assert all(set(ids[r].tolist()) <= set(left[r % 5]) | {-1} for r in range(20))
    assert all(int((ids[r] >= 0).sum()) == min(k, len(left[r % 5])) for r in range(20))


def test_more_rows_than_a_launch_takes():
    flat = F()
    nq, n = 33001, 37
    x, q = rows(n, 48, 1).cuda(), rows(nq, 48, 2).cuda()
    table = flat.FlatTable(x, metric="l2")
    s = flat.scores(table, q)
    bias = rows(1, n, 3).cuda()
    seen = torch.randint(-1, n, (nq, 3), dtype=torch.int32, generator=torch.Generator().manual_seed(4)).cuda()
    rep = torch.linspace(1, 2, nq).cuda()
    t = flat.adjust(s, bias=bias, seen=seen, repetition=rep)
    v, i = flat.topk(t, 4)
    found = flat.search(table, q, 4, bias=bias, seen=seen, repetition=rep)
    assert torch.equal(found[0], v) and torch.equal(found[1], i)
    for part in (slice(0, 70), slice(32700, 32800), slice(32960, nq)):
        sp = flat.scores(table, q[part])
        assert torch.equal(sp, s[part])
        tp = flat.adjust(sp, bias=bias, seen=seen[part], repetition=rep[part].contiguous())
        assert torch.equal(tp, t[part])
        assert torch.equal(flat.topk(tp, 4)[1], i[part])
    want = topk_plain(scores32(x.cpu(), q[-50:].cpu(), "l2"), 4)
    assert torch.equal(flat.topk(s[-50:], 4)[1].cpu(), want[1])


def test_offsets_beyond_32_bits():
    """2.4e9 scores of 16 bits, codes of 3.8e9 bytes: the ends of the table and of the matrix against a table of the ends"""
    flat = F()
    if torch.cuda.get_device_properties(0).total_memory < 64 << 30:
        pytest.skip("needs 64 GB")
    n, nq, end = 60_000_001, 40, 1000
    x = torch.randn((n, 16), generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    q = rows(nq, 16, 2).cuda()
    table, tail = flat.FlatTable(x, metric="l2"), flat.FlatTable(x[-end:], metric="l2")
    del x
    s = flat.scores(table, q, dtype=torch.float16)
    want = flat.scores(tail, q, dtype=torch.float16)
    assert torch.equal(s[:, -end:], want)
    s.clamp_(max=0)
    s[-1, -1], s[-1, 0], s[0, n // 2] = 5, 4, 3
    values, ids = flat.topk(s, 2)
    assert values[-1].tolist() == [5, 4] and ids[-1].tolist() == [n - 1, 0] and ids[0, 0] == n // 2
    bits = torch.full(((n + 31) // 32,), -1, dtype=torch.int32, device="cuda")
    bits[-1] = 0  # the last record is alone in its word
    flat.adjust(s, allow=bits, out=s)
    assert s[:, -1].eq(NEG).all() and flat.topk(s, 1)[1][-1] == 0
    del s
    f = flat.scores(table, q[-17:])  # (17, n) of 32 bits: 4.1e9 bytes
    found = flat.search(table, q[-17:], 5)
    want = flat.topk(f, 5)
    assert torch.equal(found[0], want[0]) and torch.equal(found[1], want[1])


@pytest.mark.parametrize("dim", [64, 200])
def test_search_with_biases_that_cancel_the_norms(dim):
    """((sum * q) * x - norm) + norm: what the additions round off decides between records"""
    flat = F()
    n = 30011
    table = flat.FlatTable(rows(n, dim, 1, scale=300.0).cuda(), metric="l2")
    q = rows(40, dim, 2, scale=1e-3).cuda()
    for bias in (-table.bias, -table.bias + 64.0, -table.bias * 1.0001):
        values, ids = flat.search(table, q, 20, bias=bias)
        v, i = flat.topk(flat.adjust(flat.scores(table, q), bias=bias), 20)
        assert torch.equal(ids, i) and torch.equal(values, v)


@pytest.mark.parametrize("dim", [64, 200])
def test_search_with_biases_that_are_no_numbers(dim):
    flat = F()
    n = 30011
    table = flat.FlatTable(rows(n, dim, 1).cuda(), metric="l2")
    q = rows(40, dim, 2).cuda()
    bias = rows(1, n, 3)[0]
    bias[::7], bias[1::5000], bias[2::11], bias[3::9000] = NEG, math.inf, math.nan, 3e38
    bias[4::13] = -3.4028234663852886e38
    for b in (bias, torch.where(bias.isinf() & (bias > 0), torch.tensor(0.0), bias)):
        values, ids = flat.search(table, q, 30, bias=b.cuda())
        v, i = flat.topk(flat.adjust(flat.scores(table, q), bias=b.cuda()), 30)
        assert torch.equal(ids, i) and torch.equal(values, v)


@pytest.mark.parametrize("dim", [64, 200])
def test_search_of_equal_products_whose_biases_cancel(dim):
    """the product is the same for all records: the roundings of the additions alone tell them apart"""
    flat = F()
    n, half = 30011, dim // 2
    g = torch.Generator().manual_seed(1)
    x = torch.ones(n, dim)
    x[:, half:] = torch.randint(-127, 128, (n, dim - half), generator=g).float()
    x[:, -1] = 127  # scale 50: codes are these numbers
    table = flat.FlatTable((50 * x).cuda(), metric="l2")
    q = torch.zeros(40, dim)
    q[:, :half] = 127 * torch.linspace(0.001, 0.01, 40)[:, None]
    values, ids = flat.search(table, q.cuda(), 20, bias=-table.bias)
    v, i = flat.topk(flat.adjust(flat.scores(table, q.cuda()), bias=-table.bias), 20)
    assert torch.equal(ids, i) and torch.equal(values, v)


# Small score matrices are searched by way of the matrix.  The scenarios above once more, with their queries repeated until the
# matrix is too large for that and the passes over the table search it.
class Repeating:
    MATRIX = 26 << 20

    def __init__(self, flat):
        self.flat = flat

    def __getattr__(self, name):
        return getattr(self.flat, name)

    def search(self, table, q, k, **a):
        nq = q.shape[0]
        times = 1 + self.MATRIX // (nq * table.n)

        def again(x):
            return x.repeat(times, *[1] * (x.dim() - 1)) if x.shape[0] == nq else x

        values, ids = self.flat.search(table, again(q), k, **{name: again(x) for name, x in a.items()})
        values, ids = values.view(times, nq, k), ids.view(times, nq, k)
        assert torch.equal(ids, ids[:1].expand_as(ids)) and torch.equal(values, values[:1].expand_as(values))
        return values[0], ids[0]


@pytest.mark.parametrize("scenario,arguments", [
    (test_search_equal_records_come_in_id_order, ()), (test_search_of_sorted_records, ()), (test_search_with_scales_far_apart, ()),
    (test_search_with_biases_that_cancel_the_norms, (64,)), (test_search_with_biases_that_cancel_the_norms, (200,)),
    (test_search_with_biases_that_are_no_numbers, (64,)), (test_search_with_biases_that_are_no_numbers, (200,)),
    (test_search_of_equal_products_whose_biases_cancel, (64,)), (test_search_of_equal_products_whose_biases_cancel, (200,)),
    (test_search_of_several_passes_with_little_left, (64,)), (test_search_of_several_passes_with_little_left, (200,))] +
    [(test_search_of_many_records, (n,)) for n in (8193, 131072, 400001)] +
    [(test_search_when_a_sample_misses_the_best, (n, every, k)) for n, every in ((30000, 8), (30000, 4), (270000, 9))
     for k in (1, 10, 256)] +
    [(test_search_of_several_passes_with_adjustments, (dim,) + c) for dim in (40, 128, 150, 256) for c in (
        (20, 9001, 1, 0, None, "rows"), (40, 20017, 100, 30, "shared", "rows"), (130, 70003, 10, 300, None, "shared"),
        (300, 33000, 256, 5, "shared", "rows"), (65, 300001, 17, 0, None, None), (33, 8200, 3, 4096, None, None))] +
    [(test_search, (64, 4099, 128, 10, metric)) for metric in ("ip", "l2")])
def test_search_scenarios_in_passes(scenario, arguments, monkeypatch):
    flat = Repeating(F())
    monkeypatch.setitem(globals(), "F", lambda: flat)
    scenario(*arguments)


def test_passes_captured_and_replayed_beside_other_streams():
    flat = F()
    n, nq = 30000, 2500  # two blocks of rows
    table = flat.FlatTable(rows(n, 200, 1).cuda(), metric="l2")
    a = cuda(adjustments(nq, n, 5, 20, "shared", "rows"))
    q = rows(nq, 200, 20).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        flat.search(table, q, 10, **a)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = flat.search(table, q, 10, **a)
    other = rows(nq, 200, 30).cuda()
    want_other = flat.topk(flat.scores(table, other), 5)
    for turn in range(4):
        q.copy_(rows(nq, 200, 100 + turn))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = flat.search(table, other, 5)
        torch.cuda.synchronize()
        want = flat.topk(flat.adjust(flat.scores(table, q), **a), 10)
        assert torch.equal(out[1], want[1]) and torch.equal(out[0], want[0])
        assert torch.equal(beside[1], want_other[1]) and torch.equal(beside[0], want_other[0])


def test_adjust_from_and_to_rows_that_lie_between_each_other():
    flat = F()
    both = rows(9, 202, 1)
    bias = rows(1, 100, 2)[0]
    for a, b in ((0, 100), (102, 1), (0, 0), (50, 50)):
        here = both.cuda()
        out = flat.adjust(here[:, a:a + 100], bias=bias.cuda(), out=here[:, b:b + 100])
        want = both.clone()
        want[:, b:b + 100] = both[:, a:a + 100] + bias
        assert torch.equal(here.cpu(), want) and out.data_ptr() == here[:, b:].data_ptr()
    import shine_amd
    with pytest.raises(shine_amd.ShineError, match="overlaps"):
        flat.adjust(here[:, :100], bias=bias.cuda(), out=here[:, 60:160])


def test_topk_of_rising_rows_many_times():
    """room is made in every turn of every workgroup: the answers do not depend on how its waves take turns"""
    n = 60000
    x = torch.arange(n, dtype=torch.float32).repeat(512, 1)
    x[1::2] = x[1::2].view(256, -1, 4)[:, :, [2, 0, 3, 1]].reshape(256, n)  # nearly rising
    x = x.cuda()
    for k in (100, 256):
        want = torch.arange(n - 1, n - 1 - k, -1, dtype=torch.float32, device="cuda").expand(512, k)
        for _ in range(40):
            values, ids = F().topk(x, k)
            assert torch.equal(values, want) and torch.equal(x.gather(1, ids.long()), want)


@pytest.mark.parametrize("nq", [33, 120])
@pytest.mark.parametrize("k", [10, 256])
def test_search_gives_the_same_answers_every_time(nq, k):
    """by way of the matrix and in passes, whose lists run full: in whatever order waves and workgroups come"""
    n = 270000
    x = rows(n, 32, 5) * 0.1
    x[:, 0] = torch.where((torch.arange(n) // 32) % 9 == 0, -1.0, 1.0)
    q = rows(nq, 32, 6) * 0.1
    q[:, 0] = 1
    a = cuda(adjustments(nq, n, 3, 40, "shared", "rows"))
    flat = F()
    table = flat.FlatTable(x.cuda())
    want = flat.topk(flat.adjust(flat.scores(table, q.cuda()), **a), k)
    s = flat.scores(table, q.cuda())
    for _ in range(40):
        assert torch.equal(flat.scores(table, q.cuda()), s)
        values, ids = flat.search(table, q.cuda(), k, **a)
        assert torch.equal(ids, want[1]) and torch.equal(values, want[0])


def test_calls_from_several_threads():
    import threading
    flat = F()
    table = flat.FlatTable(rows(60000, 64, 1).cuda(), metric="l2")
    qs = [rows(nq, 64, nq).cuda() for nq in (3, 40, 500, 900)]
    want = [flat.search(table, q, 20) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                values, ids = flat.search(table, qs[i], 20)
                v, j = flat.topk(flat.scores(table, qs[i]), 20)
                if not (torch.equal(values, want[i][0]) and torch.equal(ids, want[i][1]) and torch.equal(v, want[i][0])
                        and torch.equal(j, want[i][1])):
                    wrong.append(i)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(qs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("nq", [40, 1400])  # by way of the matrix, and in passes
@pytest.mark.parametrize("dim", [32, 200])
def test_search_of_records_whose_scales_were_changed(dim, nq):
    """scales of 0 and below 0 beside codes that stay: the scores are those of the changed scales"""
    flat = F()
    n = 20000
    q = rows(nq, dim, 4).cuda()
    bias = torch.full((n,), -100.0)
    bias[::200] = 0  # the answers
    for scale in (0.0, -0.0, -1e-3):
        table = flat.FlatTable(rows(n, dim, 3).cuda())
        table.scales[::200] = scale
        values, ids = flat.search(table, q, 10, bias=bias.cuda())
        v, i = flat.topk(flat.adjust(flat.scores(table, q), bias=bias.cuda()), 10)
        assert (i % 200 == 0).all() and torch.equal(ids, i) and torch.equal(values, v)
    x = rows(n, dim, 3)
    x[::200] = 0  # no codes either
    table = flat.FlatTable(x.cuda())
    values, ids = flat.search(table, q, 10, bias=bias.cuda())
    assert torch.equal(ids.cpu(), (torch.arange(10) * 200).int().expand(nq, 10)) and (values == 0).all()


@pytest.mark.parametrize("nq", [40, 1400])
def test_search_of_a_record_whose_biases_add_up_to_infinity(nq):
    """The table's bias and the call's are added to the score one after the other: with u = 2^104 the product is (2^24 - 1) u, the
    largest number, adding -(1.5 * 2^22 + 1.5) u ends halfway between two numbers and goes up to the even one, and what is left is
    what the second bias takes off.  The score is 0, far above the others, though the biases' sum is -infinity."""
    flat = F()
    n, j, unit = 20000, 7777, 2.0 ** 104
    first = (1.5 * 2 ** 22 + 1.5) * unit
    second = (2.0 ** 24 - 0.5) * unit - first
    table = flat.FlatTable(rows(n, 32, 1).cuda(), metric="l2")
    table.codes[j] = 0
    table.codes[j, 1] = 64
    table.scales[j] = torch.finfo(torch.float32).max / 64
    table.bias[j] = -first
    bias = torch.full((n,), -1000.0)
    bias[j] = -second
    q = torch.ones(nq, 32)
    q[:, 0] = 127  # scale 1, codes 127 and 1
    s = flat.adjust(flat.scores(table, q.cuda()), bias=bias.cuda())
    assert (s[:, j] == 0).all() and table.bias[j].item() == -first and bias[j].item() == -second
    assert (table.bias[j] + bias.cuda()[j]).item() == NEG
    values, ids = flat.search(table, q.cuda(), 10, bias=bias.cuda())
    v, i = flat.topk(s, 10)
    assert (i[:, 0] == j).all() and torch.equal(ids, i) and torch.equal(values, v)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim,unit", [(4000, 96, True), (700, 200, False), (50, 7, False)])
def test_distances_of_queries_as_they_are(n, dim, unit, dtype):
    """|q^ - x^|^2 between the rows that the codes stand for, never below 0, for queries that were not quantised before.

    With H = (|q^|^2 + |x^|^2) / 2 >= |<q^, x^>|: the product's three roundings and each half norm's three come to 6 u32 H, the
    score's addition and the last one, of at most 2 H each, to 4 u32 H, and twice all of it is 20 u32 H."""
    flat = F()
    x = rows(n, dim, dim)
    m = min(n, 60)
    q = x[:m] + torch.linspace(-0.3, 0.7, m).clamp_min(0)[:, None] * rows(m, dim, 2)  # records themselves, and rows farther away
    if unit:
        x, q = torch.nn.functional.normalize(x), torch.nn.functional.normalize(q)
    x, q = x.to(dtype), q.to(dtype)
    table = flat.FlatTable(x.cuda(), metric="l2")
    values, ids = flat.search(table, q.cuda(), 5)
    d = table.distances(values, q.cuda())
    assert d.dtype == torch.float32 and (d >= 0).all()
    xc, xs = codes64(x)
    qc, qs = codes64(q)
    xd, qd = xc * xs[:, None], qc * qs[:, None]
    found = xd[ids.cpu().long()]
    want = (qd[:, None] - found).square().sum(2)
    half = (qd.square().sum(1)[:, None] + found.square().sum(2)) / 2
    assert ((d.cpu().double() - want).abs() <= 20.01 * U32 * half).all()
    assert torch.equal(table.distances(values.cpu(), q), d.cpu())
    whole = table.distances(flat.scores(table, q.cuda()), q.cuda())
    assert torch.equal(whole.gather(1, ids.long()), d)


def test_distances_of_places_without_an_answer():
    flat = F()
    table = flat.FlatTable(rows(3, 16, 1).cuda(), metric="l2")
    q = rows(4, 16, 2)
    q[1, 3], q[2, 5] = math.nan, math.inf
    values, ids = flat.search(table, q.cuda(), 5)
    d = table.distances(values, q.cuda())
    assert torch.equal(d.isposinf(), ids < 0) and d[[0, 3], :3].isfinite().all()
    with pytest.raises(ValueError, match="dim 15"):
        table.distances(values, q[:, :15].cuda())
    with pytest.raises(ValueError, match="inner products"):
        flat.FlatTable(rows(3, 16, 1).cuda()).distances(values, q.cuda())


def test_adjustments_that_require_gradients_are_refused():
    flat = F()
    x = rows(20, 32, 1).cuda()
    table = flat.FlatTable(x)
    seen = torch.zeros((20, 1), dtype=torch.int32, device="cuda")
    for name, like in (("bias", torch.zeros(20)), ("bias", torch.zeros(20, 20)), ("repetition", torch.ones(20)),
                       ("frequency", torch.ones(20)), ("presence", torch.ones(20))):
        a = {name: like.cuda().requires_grad_()}
        if name != "bias":
            a["seen"] = seen
        with pytest.raises(ValueError, match=f"{name} requires a gradient"):
            flat.adjust(flat.scores(table, x), **a)
        with pytest.raises(ValueError, match=f"{name} requires a gradient"):
            flat.search(table, x, 3, **a)
        with torch.no_grad():
            want = flat.adjust(flat.scores(table, x), **{k: v.detach() for k, v in a.items()})
            assert torch.equal(flat.adjust(flat.scores(table, x), **a), want)
            assert torch.equal(flat.search(table, x, 3, **a)[1], flat.topk(want, 3)[1])


@pytest.mark.parametrize("nq,n", [(3, 700), (40, 9001), (2100, 20000)])
def test_a_history_shared_by_all_rows(nq, n):
    flat = F()
    table = flat.FlatTable(rows(n, 64, 1).cuda(), metric="l2")
    q = rows(nq, 64, 2).cuda()
    s = flat.scores(table, q)
    a = cuda(adjustments(nq, n, 3, 50))
    seen = a.pop("seen")[0]
    for one in (seen, seen[None], seen[:1], seen[:0]):
        each = one.reshape(1, -1).repeat(nq, 1)
        want = flat.adjust(s, seen=each, **a)
        assert torch.equal(flat.adjust(s, seen=one, **a), want)
        assert torch.equal(flat.adjust(s, seen=one.reshape(1, -1).expand(nq, -1), **a), want)
        v, i = flat.topk(want, 20)
        values, ids = flat.search(table, q, 20, seen=one, **a)
        assert torch.equal(ids, i) and torch.equal(values, v)


def hip_runtime():
    """the HIP runtime that this process has loaded"""
    maps = open("/proc/self/maps").read().split()
    return C.CDLL(next(path for path in maps if "libamdhip64.so" in path))


def test_errors_are_reported_once_and_by_the_call_that_met_them():
    from shine_amd import _lib as L
    flat = F()
    x = rows(20, 32, 1).cuda()
    want, scale = codes64(x.cpu())
    codes, scales = torch.empty((20, 64), dtype=torch.int8, device="cuda"), torch.empty(20, device="cuda")
    quantize = L.lib().shine_flat_quantize
    stream = torch.cuda.current_stream().cuda_stream

    def call(gpu):
        return quantize(gpu, x.data_ptr(), 0, 20, 32, 32, codes.data_ptr(), scales.data_ptr(), None, stream)

    assert call(torch.cuda.device_count()) == L.ERR_HIP  # no such device
    assert call(0) == L.OK
    assert call(torch.cuda.device_count()) == L.ERR_HIP
    assert (x + 1).shape == x.shape  # nor do others meet it
    # what another call left behind is not flat scoring's, to report or to clear
    hip = hip_runtime()
    table = flat.FlatTable(x, metric="l2")
    rc = hip.hipSetDevice(torch.cuda.device_count())
    assert rc != 0
    try:
        assert call(0) == L.OK
        got = L.lib().shine_flat_topk(0, x.data_ptr(), 0, 20, 32, 32, 1, scales.data_ptr(), codes.data_ptr(), None, 0, stream)
    finally:
        left = hip.hipGetLastError()
    assert got == L.OK and left == rc
    assert call(0) == L.OK
    assert torch.equal(codes[:, :32].cpu().double(), want) and torch.equal(scales.cpu().double(), scale)
    assert (flat.search(table, x, 1)[1][:, 0] >= 0).all()


def test_more_rows_or_shown_ids_than_32_bits_count_are_refused():
    """they were taken modulo 2^32; nothing here is read or written"""
    import shine_amd
    flat = F()
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GB")
    many = torch.empty((2 ** 32 + 1, 1), dtype=torch.float16, device="cuda")
    table = flat.FlatTable(rows(5, 1, 1).cuda())
    for call in (lambda: flat.topk(many, 1), lambda: flat.adjust(many, out=many), lambda: flat.search(table, many, 1),
                 lambda: flat.scores(table, many)):
        with pytest.raises(ValueError, match="at most 4294967295 rows"):
            call()
    del many
    ids = torch.empty((1, 2 ** 32 + 3), dtype=torch.int32, device="cuda")
    for call in (lambda: flat.adjust(rows(2, 10, 1).cuda(), seen=ids), lambda: flat.search(table, rows(2, 1, 1).cuda(), 1, seen=ids)):
        with pytest.raises(shine_amd.ShineError, match="65535"):
            call()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,n,dim", [(3, 400, 96), (40, 1000, 200), (33, 500, 768)])
def test_scores_are_near_the_products_of_the_rows_themselves(nq, n, dim, dtype):
    """A component is within half a scale of its code's: with q^ = q + d and x^ = x + e,
    |<q^, x^> - <q, x>| <= |q|_1 sx / 2 + |x|_1 sq / 2 + dim sq sx / 4, and three roundings of the product."""
    x, q = rows(n, dim, 1, dtype), rows(nq, dim, 2, dtype)
    s = F().scores(F().FlatTable(x.cuda()), q.cuda()).cpu().double()
    x, q = x.double(), q.double()
    sx, sq = (codes64(r)[1] for r in (x, q))
    bound = q.abs().sum(1)[:, None] * sx / 2 + sq[:, None] * x.abs().sum(1) / 2 + dim * sq[:, None] * sx / 4
    assert ((s - q @ x.T).abs() <= bound + 3.01 * U32 * s.abs()).all()
