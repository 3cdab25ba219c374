"""GPU: where the block operators' ranges end — values that are not numbers in rows a key is hidden from, weights and gradients at the ends of
binary16, log-sum-exps of more keys than a call's, strides and sizes beyond the usual ones — against their definitions in binary64."""
import numpy as np
import pytest
import torch

import blocks_ref as ref
import test_gpu_blocks as base
from test_gpu_blocks import SENTINEL, Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def blocks(gp):
    from pygpann import blocks
    return blocks


def formula(p, b, t, h, heads, vis, out, lse, probes):
    """A query row's gradients as the header's formula has them, from a given out and lse, and their bounds without the rounding of the results.

    E = 2^-24, u = half a step of the type, s = half the smallest step of binary16 (2^-25) or 0.  A logit is off by (d + 4) E a, a = |scale| sum |q_i k_i| at most, and
    a weight by w = 2 (d + 4) E a + 8 E + 4 E |lse| of itself (exponent's argument and lse * log2 e); dp and delta by (d + 2) E of the sums of their terms' sizes.
    delta may be corrected for the rounding of out: by no more than 1.25 (u sum |dout out| + s sum |dout|), what that rounding can have come to and a quarter more.
    p and ds are rounded once, to u of themselves or s; sums of n terms in binary32 add n E of the terms' sizes."""
    u, s, d = ref.U[p.dtype], 2.0 ** -25 if p.dtype == "fp16" else 0.0, p.dim
    rows = ref.rows_of(probes[b, t, h], p.bs, p.nblk, vis)
    q, k, v, do = p.q64[b, t, heads], p.k64[b, rows, h], p.v64[b, rows, h], p.do64[b, t, heads]
    o, l = out[b, t, heads], lse[b, t, heads]
    if len(rows) == 0:
        return rows, np.zeros_like(q), None, None, np.zeros_like(q), None, None
    a = abs(p.scale) * (np.abs(q) @ np.abs(k).T)
    w = 2 * (d + 4) * ref.E * a + 8 * ref.E + 4 * ref.E * np.abs(l)[:, None]
    pr = np.exp(p.scale * (q @ k.T) - l[:, None])
    delta = (do * o).sum(1, keepdims=True)
    ds = pr * (do @ v.T - delta)
    off = 1.25 * (u * (np.abs(do) * np.abs(o)).sum(1, keepdims=True) + s * np.abs(do).sum(1, keepdims=True))
    dp_err = (d + 2) * ref.E * (np.abs(do) @ np.abs(v).T + (np.abs(do) * np.abs(o)).sum(1, keepdims=True)) + off
    ds_err = pr * (1 + w) * dp_err + (w + u + 2 * ref.E) * np.abs(ds) + s
    n = len(rows)
    return (rows, p.scale * (ds @ k), p.scale * (ds.T @ q), pr.T @ do, abs(p.scale) * ((ds_err + n * ref.E * np.abs(ds)) @ np.abs(k)),
            abs(p.scale) * (ds_err.T @ np.abs(q)), ((w + u) * pr).T @ np.abs(do))


def check_gradients(p, probes=None, but=(), hidden=None):
    """dq, dk and dv against the formula.  `but`: query rows (sequence, row) that take no part; `hidden` [batch][key][kv head]: the keys whose dk, dv are compared"""
    u, tiny = ref.U[p.dtype], 2.0 ** -25 if p.dtype == "fp16" else 0.0
    probes = p.probes_np if probes is None else probes
    out, lse = p.out.double().cpu().numpy(), p.lse.double().cpu().numpy()
    got = {x: getattr(p, x).double().cpu().numpy() for x in ("dq", "dk", "dv")}
    want, tol = ({x: np.zeros(y.shape) for x, y in got.items()} for _ in range(2))
    size, terms = {x: np.zeros(got[x].shape) for x in ("dk", "dv")}, np.zeros(got["dk"].shape[:3])
    take = {"dq": np.ones(got["dq"].shape, bool), "dk": np.ones(got["dk"].shape, bool), "dv": np.ones(got["dv"].shape, bool)}
    for b, t, h, heads, vis in p.rows():
        if (b, t) in but:
            take["dq"][b, t] = False
            continue
        rows, dq, dk, dv, eq, ek, ev = formula(p, b, t, h, heads, vis, out, lse, probes)
        want["dq"][b, t, heads], tol["dq"][b, t, heads] = dq, eq
        if len(rows):
            for x, y, e in (("dk", dk, ek), ("dv", dv, ev)):
                want[x][b, rows, h] += y
                tol[x][b, rows, h] += e
                size[x][b, rows, h] += np.abs(y) + e
            terms[b, rows, h] += p.G
    for x in ("dk", "dv"):
        tol[x] += (terms[..., None] + 8) * ref.E * size[x]       # binary32 sums over query rows and heads
        if hidden is not None:
            take[x] &= hidden[..., None]
    for x in got:
        bound = tol[x] + u * (np.abs(want[x]) + tol[x]) + tiny
        over = (np.abs(want[x]) + tol[x] >= 65520) & (got[x] == np.copysign(np.inf, want[x])) if p.dtype == "fp16" else False      # rounds to an infinity there
        with np.errstate(invalid="ignore"):
            bad = ~((np.abs(got[x] - want[x]) <= bound) | over) & take[x]
        assert not bad.any(), (x, np.argwhere(bad)[:4], got[x][bad][:4], want[x][bad][:4], bound[bad][:4])
        assert take[x].any()


def not_seen_by(p, rows):
    """[batch][key][kv head]: keys that none of these query rows looks at"""
    hidden = np.ones(p.k64.shape[:3], bool)
    for b, t, h, heads, vis in p.rows():
        if (b, t) in rows:
            hidden[b, ref.rows_of(p.probes_np[b, t, h], p.bs, p.nblk, vis), h] = False
    return hidden


# ---- gradients: rows that a key is hidden from -------------------------------------------------------------------------------------------------
HIDDEN = [dict(), dict(dim=128, bs=64), dict(dim=96, bs=16, dtype="fp16"), dict(dim=192, dtype="fp16", bs=48), dict(dim=256, bs=128), dict(q_heads=40, kv_heads=2, bs=32, dtype="fp16"),
          dict(q_heads=1, kv_heads=1, bs=256, scale=-0.2), dict(causal=False, bs=64), dict(q_rows=300, kv_rows=320, kv_len=[310], q_heads=32, kv_heads=1, bs=64, middle=(250, 262))]


@pytest.mark.parametrize("kw", HIDDEN, ids=str)
@pytest.mark.parametrize("where", ["middle", "last"])
def test_rows_that_are_not_numbers_leave_the_keys_alone_that_they_do_not_see(blocks, kw, where):
    """an infinity in one query row's dout and a NaN in another's q, both in the middle of a block, or an infinity in the last row of all: the keys behind them in their
    blocks, and the cache's rows behind the sequence, have the gradients of the other query rows"""
    kw = dict(kw)
    middle = kw.pop("middle", (5, 9))
    kw = {**dict(seed=81, batch=1, q_rows=40, kv_rows=160, kv_len=[150], nprobe=3), **kw}
    bs, n = kw.get("bs", 32), kw["kv_len"][0]
    probes = np.random.default_rng(5).integers(-1, -(-kw["kv_rows"] // bs) + 1, size=(1, kw["q_rows"], kw.get("kv_heads", 2), 3))
    probes[..., 0], probes[..., 1] = (n - 1) // bs, max(0, (n - 1) // bs - 1)
    for t in middle:
        probes[0, t, :, 2] = (n - kw["q_rows"] + t) // bs          # its own block
    p = Problem(blocks, probes=probes, **kw)
    if where == "last":
        rows = [(0, p.q_rows - 1)]
        p.dout[0, -1, -1, 0] = -float("inf")
    else:
        rows = [(0, t) for t in middle]
        p.dout[0, middle[0], :, 3] = float("inf")
        p.q[0, middle[1], :, 7] = float("nan")
    p.attend()
    p.backward()
    torch.cuda.synchronize()
    check_gradients(p, but=rows, hidden=not_seen_by(p, rows))
    assert (p.dk[0, n:] == 0).all() and (p.dv[0, n:] == 0).all()
    if where == "middle":         # as the formula has it
        assert torch.isnan(p.dq[0, middle[1]]).all()
        seen = torch.from_numpy(~not_seen_by(p, rows[1:])).cuda()
        assert torch.isnan(p.dk[seen]).all() and torch.isnan(p.dv[seen]).all()
    first = [x.clone() for x in (p.dq, p.dk, p.dv)]
    p.backward()
    for x, y in zip(first, (p.dq, p.dk, p.dv)):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


# ---- gradients: the ends of binary16 -----------------------------------------------------------------------------------------------------------
def scaled(p, **factors):
    """tensors multiplied by powers of two (exactly)"""
    for name, f in factors.items():
        x = getattr(p, name)
        x.mul_(f)
        wide = {"q": "q64", "k": "k64", "v": "v64", "dout": "do64"}[name]
        setattr(p, wide, getattr(p, wide) * f)


@pytest.mark.parametrize("kw", [dict(), dict(dim=128, bs=16), dict(dim=192), dict(dim=256, bs=32), dict(q_heads=24, kv_heads=1, bs=64), dict(dim=96, q_rows=60, kv_rows=60, bs=16, kv_len=[60, 33])],
                         ids=str)
def test_gradients_whose_terms_binary16_cannot_hold(blocks, kw):
    """|ds| above 65504, dq, dk and dv within the type: dout of order 2^13 against values of order 4, a scale of 0.03"""
    p = Problem(blocks, **{**dict(seed=82, q_rows=5, kv_rows=64, kv_len=[3, 9], bs=16, dtype="fp16", scale=0.03), **kw})
    p.probes_np[...] = np.arange(4)
    p.probes.copy_(torch.from_numpy(p.probes_np))
    scaled(p, v=4.0, dout=2.0 ** 13)
    p.attend()
    p.backward()
    torch.cuda.synchronize()
    check_gradients(p)
    most = 0.0
    for b, t, h, heads, vis in p.rows():
        rows = ref.rows_of(p.probes_np[b, t, h], p.bs, p.nblk, vis)
        if len(rows):
            lse, pr, _ = ref.softmax_rows(p.q64[b, t, heads], p.k64[b, rows, h], p.scale)
            dp = p.do64[b, t, heads] @ p.v64[b, rows, h].T
            most = max(most, np.abs(pr * (dp - (pr * dp).sum(1, keepdims=True))).max())
    assert most > 65520          # the case is what it says


@pytest.mark.parametrize("kw", [dict(), dict(dim=128, bs=32), dict(dim=256, bs=128), dict(q_rows=300, kv_rows=2000, q_heads=32, kv_heads=1, bs=256, nprobe=8)], ids=str)
def test_values_gradients_of_weights_that_binary16_cannot_hold(blocks, kw):
    """one key has nearly all the weight of every row, the others about 2^-26 each: their dv is a sum of such"""
    kw = {**dict(seed=83, batch=1, q_rows=64, kv_rows=1000, q_heads=4, kv_heads=2, bs=64, nprobe=16, dtype="fp16", strength=0.5), **kw}
    p = Problem(blocks, **kw)
    p.probes_np[...] = np.arange(p.nprobe)
    p.probes.copy_(torch.from_numpy(p.probes_np))
    for x, y in ((p.q, p.q64), (p.k, p.k64)):
        x[..., 0], y[..., 0] = 0, 0
    p.q[..., 0], p.q64[..., 0] = 16, 16
    lift = 18.0 / (16 * p.scale)            # (e^-18 = 2^-26; the type's nearest number)
    p.k[:, 0, :, 0] = lift
    p.k64[:, 0, :, 0] = float(p.k[0, 0, 0, 0])
    scaled(p, dout=2.0 ** 11)
    p.attend()
    p.backward()
    torch.cuda.synchronize()
    check_gradients(p)
    assert (p.dv != 0).float().mean() > 0.5


# ---- gradients from the out and lse of more keys than the call's -----------------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(), dict(dim=128, bs=64, kv_rows=400, dtype="fp16"), dict(dim=192, bs=16), dict(dim=256, q_heads=20, kv_heads=1), dict(causal=False, q_heads=2, kv_heads=2)], ids=str)
def test_gradients_of_two_calls_whose_attention_was_joined(blocks, kw):
    """two probe lists, their outs and log-sum-exps joined, each call's gradients from the joined ones: the header's formula for either"""
    p = Problem(blocks, **{**dict(seed=84, batch=2, q_rows=40, kv_rows=150, nprobe=8), **kw})
    lists = [np.full_like(p.probes_np, -1) for _ in range(2)]
    for j in range(min(16, p.nblk)):
        lists[j % 2][..., j // 2] = j
    outs, lses = [], []
    for probes in lists:
        p.probes.copy_(torch.from_numpy(probes))
        p.attend()
        outs.append(p.out.double())
        lses.append(p.lse.double())
    lse = torch.logaddexp(*lses)
    out = sum((l - lse).exp().nan_to_num(0.0)[..., None] * o for l, o in zip(lses, outs))
    p.lse.copy_(lse)
    p.out.copy_(out)
    for probes in lists:
        p.probes.copy_(torch.from_numpy(probes))
        p.backward()
        torch.cuda.synchronize()
        check_gradients(p, probes=probes)


# ---- strides and sizes --------------------------------------------------------------------------------------------------------------------------
def test_gradients_of_heads_that_lie_as_far_apart_as_a_layout_allows(blocks):
    """q, out and their gradients with a head stride of 2^31 elements"""
    p = Problem(blocks, seed=85, batch=1, q_rows=20, kv_rows=90, q_heads=2, kv_heads=1)
    far = 2 ** 31
    stride = (2 ** 33, 64, far, 1)
    wide = {}
    for name in ("q", "out", "dout", "dq"):
        wide[name] = torch.empty(far + 20 * 64, dtype=torch.bfloat16, device="cuda")
    place = lambda name: torch.as_strided(wide[name], (1, 20, 2, 64), stride)
    place("q").copy_(p.q)
    place("dout").copy_(p.dout)
    L = blocks.Layout(1, 20, 90, 2, 1, 64, 32, scale=p.scale, q_stride=stride[:3], out_stride=stride[:3], k_stride=p.k.stride()[:3], v_stride=p.v.stride()[:3])
    p.L = L
    tensors = {x: getattr(p, x) for x in ("q", "dout")}
    p.q, p.out, p.dout, p.dq = (place(x) for x in ("q", "out", "dout", "dq"))
    p.dk, p.dv = torch.empty_like(p.k), torch.empty_like(p.v)
    p.attend()
    p.backward_call()
    torch.cuda.synchronize()
    p.check_attend()
    p.check_backward()
    assert torch.equal(p.q, tensors["q"]) and torch.equal(p.dout, tensors["dout"])


def test_an_eviction_that_could_keep_far_more_than_there_is(blocks):
    """keep = 2^24 of 64 rows: a launch's work is that of the rows"""
    p = Problem(blocks, seed=86, batch=1, kv_rows=64, kv_heads=1, q_heads=1)
    keep = 1 << 24
    mass = torch.rand(1, 1, 64, device="cuda")
    rows, mass_out = torch.full((1, 1, keep), -5, dtype=torch.int32, device="cuda"), torch.full((1, 1, keep), SENTINEL, device="cuda")
    count = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    call = lambda: blocks.evict(p.L, None, None, mass.data_ptr(), keep, rows.data_ptr(), count.data_ptr(), mass_out=mass_out.data_ptr(), **p.space)
    call()
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    call()
    end.record()
    torch.cuda.synchronize()
    assert count.item() == 64 and rows[0, 0, :64].tolist() == list(range(64)) and (rows[0, 0, 64:] == -5).all()
    assert torch.equal(mass_out[0, 0, :64], mass[0, 0]) and (mass_out[0, 0, 64:] == SENTINEL).all()
    assert start.elapsed_time(end) < 3.0      # ms; two launches take hundredths of one, a loop over 2^24 slots by 512 threads hundreds


@pytest.mark.parametrize("kw", [dict(keep=20000, kv_rows=33000, ties=True), dict(keep=500, kv_rows=70000, ties=True, first=4, last=100), dict(keep=33000, kv_rows=70000, kv_len=[70000, 32769])], ids=str)
def test_evict_from_sequences_that_do_not_fit_lds(blocks, kw):
    base.test_evict(blocks, kw)


@pytest.mark.parametrize("kw", [dict(q_rows=2100), dict(q_rows=4200, dim=128, q_heads=3), dict(q_rows=2500, bs=80, paged=True, kv_len=[333])], ids=str)
def test_weigh_of_more_query_rows_than_a_wavefront_lists_at_a_time(blocks, kw):
    base.test_weigh(blocks, {**dict(batch=1, kv_rows=350, q_heads=2, kv_heads=1, bs=64, nprobe=3), **kw}, True)


@pytest.mark.parametrize("kw", [dict(q_rows=1, kv_rows=20000), dict(q_rows=2, kv_rows=80000, nprobe=64), dict(q_rows=5, kv_rows=80000, dim=96, dtype="fp16", kv_len=[80000, 65600]),
                                dict(q_rows=1, kv_rows=16 * 16384, nprobe=9, batch=1)], ids=str)
def test_route_over_more_blocks_than_registers_hold(blocks, kw):
    base.test_route(blocks, {**dict(bs=16, nprobe=20, q_heads=2, kv_heads=1), **kw})


@pytest.mark.parametrize("kw", [dict(q_rows=2100, kv_rows=2100, bs=64), dict(q_rows=17000, kv_rows=400, bs=128, causal=False), dict(q_rows=17000, kv_rows=17000, bs=256, nprobe=2, dtype="fp16"),
                                dict(q_rows=4500, kv_rows=4500, bs=16, dim=192, kv_len=[4400])], ids=str)
def test_backward_of_more_query_rows_than_are_listed_at_a_time(blocks, kw):
    p = Problem(blocks, **{**dict(seed=87, batch=1, q_heads=1, kv_heads=1, nprobe=3), **kw})
    p.attend()
    p.backward()
    torch.cuda.synchronize()
    p.check_attend()
    p.check_backward()


# ---- layouts of other orders --------------------------------------------------------------------------------------------------------------------
def spread(p, out_order=(0, 2, 1, 3)):
    """q, k and v become slices of one packed tensor each with a gap behind every row, out, dout and their like [sequence][head][row][dim]; what is behind the
    sequences' ends, and the gaps, hold NaN"""
    def gapped(x, extra):
        rows = torch.full((*x.shape[:2], x.shape[2] + extra, x.shape[3] + 8), float("nan"), dtype=x.dtype, device=x.device)
        view = rows[:, :, extra:, 8:]
        view.copy_(x)
        return view
    def turned(x):
        y = torch.empty([x.shape[i] for i in out_order], dtype=x.dtype, device=x.device).permute(out_order)
        return y.copy_(x)
    p.q, p.k, p.v = gapped(p.q, 3), gapped(p.k, 1), gapped(p.v, 2)
    p.out, p.dout = turned(p.out), turned(p.dout)
    for b in range(p.batch):
        p.dout[b, p.m[b]:] = float("nan")
    p.L = p.blocks.Layout(p.batch, p.q_rows, p.kv_rows, p.q_heads, p.kv_heads, p.dim, p.bs, dtype=p.dtype, causal=p.causal, scale=p.scale,
                          q_len=None if p.ql_t is None else p.ql_t.data_ptr(), kv_len=None if p.kv_t is None else p.kv_t.data_ptr(),
                          q_stride=p.q.stride()[:3], k_stride=p.k.stride()[:3], v_stride=p.v.stride()[:3], out_stride=p.out.stride()[:3])


LAYOUTS = [dict(), dict(q_rows=1, kv_rows=700, bs=64, dim=128), dict(q_rows=1, batch=5, bs=80, dim=256, nprobe=9), dict(bs=112, q_heads=14, dim=96, dtype="fp16"),
           dict(bs=208, kv_rows=900, dim=192), dict(bs=240, kv_rows=900, q_rows=60, q_heads=3, kv_heads=1, kv_len=[777, 3], q_len=[60, 9]), dict(bs=80, dim=256, dtype="fp16", q_rows=30),
           dict(batch=16, q_rows=40, q_heads=32, kv_heads=8, bs=144, kv_rows=300, dim=128, q_len=[40, 0] * 8), dict(batch=16, kv_heads=16, q_heads=256, q_rows=20, bs=176, kv_rows=400)]


@pytest.mark.parametrize("kw", LAYOUTS, ids=str)
def test_tensors_of_other_orders_and_strides(blocks, kw):
    p = Problem(blocks, **{**dict(seed=91), **kw})
    spread(p)
    p.attend()
    torch.cuda.synchronize()
    p.check_attend()
    lse = p.lse.clone()
    p.out.fill_(SENTINEL)
    blocks.attend(p.L, p.q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(), p.probes.data_ptr(), p.nprobe, p.out.data_ptr(), **p.space)      # no lse wanted
    torch.cuda.synchronize()
    p.check_attend()
    for b in range(p.batch):
        p.lse[b, p.m[b]:] = float("nan")
        p.out[b, p.m[b]:] = float("nan")
    for name in ("q", "k", "v"):
        x = getattr(p, name)
        base_tensor = torch.full((x.shape[0] * x.stride(0),), SENTINEL, dtype=x.dtype, device="cuda")
        setattr(p, "d" + name, torch.as_strided(base_tensor, x.shape, x.stride()))
    p.backward_call()
    torch.cuda.synchronize()
    check_gradients(p)
    p.check_backward()
    for name in ("q", "k", "v"):           # the gaps are nobody's
        x = getattr(p, "d" + name)
        whole = torch.as_strided(x, (x.shape[0] * x.stride(0),), (1,), 0).clone()
        torch.as_strided(whole, x.shape, x.stride()).fill_(SENTINEL)
        assert (whole == SENTINEL).all()
    assert torch.equal(lse[p.lse == p.lse], p.lse[p.lse == p.lse])


@pytest.mark.parametrize("kw", [dict(), dict(bs=80, dim=256, kv_rows=333, q_rows=20), dict(kv_len=[150, 61], nprobe=3, dim=96, dtype="fp16", q_rows=40)], ids=str)
def test_routing_weights_and_eviction_of_other_orders_and_strides(blocks, kw):
    p = Problem(blocks, **{**dict(seed=92, nprobe=3), **kw})
    spread(p)
    s = torch.full((p.batch, p.kv_heads, p.nblk, p.dim), SENTINEL, device="cuda")
    blocks.summarize(p.L, p.k.data_ptr(), s.data_ptr())
    probes = torch.full_like(p.probes, 12345)
    blocks.route(p.L, p.q.data_ptr(), s.data_ptr(), p.nprobe, probes.data_ptr(), first=1, last=1, **p.space)
    got, cen = probes.cpu().numpy(), s.cpu().numpy()
    for b, t, h, heads, vis in p.rows():
        assert np.array_equal(cen[b, h, :-(-p.n[b] // p.bs)], ref.summarize(p.k64[b, :, h], p.n[b], p.bs))
        assert np.array_equal(got[b, t, h], ref.route(p.q64[b, t, heads], cen[b, h], p.bs, vis, p.nprobe, 1, 1)), (b, t, h)
    p.attend()
    mass = torch.zeros(p.batch, p.kv_heads, p.kv_rows, device="cuda")
    blocks.weigh(p.L, p.q.data_ptr(), p.k.data_ptr(), p.probes.data_ptr(), p.nprobe, p.lse.data_ptr(), mass.data_ptr(), mass.data_ptr(), **p.space)
    weights, sums = mass.cpu().numpy(), np.zeros((p.batch, p.kv_heads))
    for b, t, h, heads, vis in p.rows():
        sums[b, h] += p.G * (len(ref.rows_of(p.probes_np[b, t, h], p.bs, p.nblk, vis)) > 0)
    assert np.allclose(weights.sum(2), sums, rtol=1e-4)          # (every head spreads a weight of 1; binary32 sums of at most 1000 terms)
    keep = 45
    rows, count = torch.full((p.batch, p.kv_heads, keep), -5, dtype=torch.int32, device="cuda"), torch.zeros(p.batch, p.kv_heads, dtype=torch.int32, device="cuda")
    both = torch.full((p.batch, p.kv_heads, 2, keep, p.dim), SENTINEL, dtype=p.k.dtype, device="cuda")          # [sequence][head][k, v][row][dim]
    k_out, v_out = (both[:, :, i].permute(0, 2, 1, 3) for i in range(2))
    blocks.evict(p.L, p.k.data_ptr(), p.v.data_ptr(), mass.data_ptr(), keep, rows.data_ptr(), count.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), first=2, last=3,
                 out_kv_stride=k_out.stride()[:3], **p.space)
    for b in range(p.batch):
        for h in range(p.kv_heads):
            want = ref.evict(weights[b, h], p.n[b], keep, 2, 3)
            c = len(want)
            assert count[b, h] == c and rows[b, h, :c].tolist() == want
            assert np.array_equal(k_out[b, :c, h].double().cpu().numpy(), p.k64[b, want, h]) and np.array_equal(v_out[b, :c, h].double().cpu().numpy(), p.v64[b, want, h])
            assert (k_out[b, c:, h] == SENTINEL).all() and (v_out[b, c:, h] == SENTINEL).all()


# ---- attention whose weights binary16 holds only in part ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(batch=1, q_rows=1), dict(batch=1, q_rows=1, dim=256, kv_heads=2), dict(batch=64, q_rows=1, kv_rows=300), dict(batch=8, q_rows=40, q_heads=16, kv_heads=8, kv_rows=400),
                                dict(batch=16, kv_heads=16, q_heads=256, q_rows=20, kv_rows=300, dim=128), dict(batch=8, q_rows=40, q_heads=32, kv_heads=8, kv_rows=300, dim=192, bs=16),
                                dict(batch=8, q_rows=40, q_heads=16, kv_heads=8, kv_rows=400, beside=True)], ids=str)
def test_attention_that_hangs_on_weights_binary16_holds_in_part(blocks, kw):
    """one key has nearly all the weight and the value 0: out is a sum over the others, whose weights are 2^-16 to 2^-20"""
    kw = {**dict(seed=95, kv_rows=1000, q_heads=4, kv_heads=2, bs=64, nprobe=16, dtype="fp16"), **kw}
    beside = kw.pop("beside", False)
    p = Problem(blocks, **kw)
    p.probes_np[...] = np.where(np.arange(p.nprobe) < p.nblk, np.arange(p.nprobe), -1)
    if beside:          # every second row sees values that are none: the others are done again by themselves
        p.probes_np[:, 1::2, :, p.nblk - 1] = -1
    p.probes.copy_(torch.from_numpy(p.probes_np))
    bits = np.linspace(16, 20, p.q_rows * p.q_heads).reshape(p.q_rows, p.q_heads)
    for x, y in ((p.q, p.q64), (p.k, p.k64)):
        x.zero_()
        y[...] = 0
    p.q[..., 0] = torch.from_numpy(bits * np.log(2) / p.scale / 64).to(p.q)
    p.q64[..., 0] = p.q[..., 0].double().cpu().numpy()
    p.k[:, 0, :, 0] = p.k64[:, 0, :, 0] = 64
    p.v.abs_().mul_(4)
    p.v[:, 0], p.v64[...] = 0, np.abs(p.v64) * 4
    p.v64[:, 0] = 0
    if beside:
        p.v[:, (p.nblk - 1) * p.bs:] = float("nan")
    p.attend()
    torch.cuda.synchronize()
    out = p.out.double().cpu().numpy()
    for b, t, h, heads, vis in p.rows():
        if not beside or t % 2:
            want, _, tol, _ = ref.attend(p.q64[b, t, heads], p.k64[b, :, h], p.v64[b, :, h], p.probes_np[b, t, h], p.bs, p.nblk, vis, p.scale, p.dtype)
            assert (np.abs(out[b, t, heads] - want) <= tol).all(), (b, t, h, np.abs(out[b, t, heads] / want - 1).max())


@pytest.mark.parametrize("kw", [dict(), dict(dim=192, bs=64), dict(q_rows=70, kv_rows=300, q_heads=16, kv_heads=1)], ids=str)
def test_gradients_of_values_near_the_smallest_of_binary16(blocks, kw):
    """values of 2^-16: the steps of out are a hundredth of it, and delta's error is told from the weights' own sum all the same.  Against the gradient at the unrounded out:
    what is left of delta's error is the sum of the ds' own rounding, u sum |ds|, the weights' in out (u sum p |dp|) and binary32's"""
    p = Problem(blocks, **{**dict(seed=96, batch=1, q_rows=40, kv_rows=150, nprobe=5, dtype="fp16"), **kw})
    p.probes_np[...] = np.arange(p.nprobe)
    p.probes.copy_(torch.from_numpy(p.probes_np))
    scaled(p, dout=2.0 ** 8)
    p.v.mul_(2.0 ** -16)
    p.v64 = p.v.double().cpu().numpy()
    p.v64[np.isnan(p.v64)] = 0
    p.attend()
    p.backward()
    torch.cuda.synchronize()
    u, got, s = ref.U["fp16"], p.dq.double().cpu().numpy(), 2.0 ** -25
    for b, t, h, heads, vis in p.rows():
        rows = ref.rows_of(p.probes_np[b, t, h], p.bs, p.nblk, vis)
        if len(rows) == 0:
            continue
        k, v, do = p.k64[b, rows, h], p.v64[b, rows, h], p.do64[b, t, heads]
        lse, pr, w = ref.softmax_rows(p.q64[b, t, heads], k, p.scale)
        dp = do @ v.T
        ds = pr * (dp - (pr * dp).sum(1, keepdims=True))
        n, away = len(rows), np.abs(k)
        each = (u + 3 * w + n * ref.E) * np.abs(ds) + (p.dim + 2) * ref.E * pr * (np.abs(do) @ np.abs(v).T) + s                  # a ds' own error
        left = each.sum(1, keepdims=True) + (u + w) * (pr * np.abs(dp)).sum(1, keepdims=True)                                  # delta's
        bound = abs(p.scale) * ((each + pr * left) @ away)
        want = p.scale * (ds @ k)
        bound += u * (np.abs(want) + bound) + s
        assert (np.abs(got[b, t, heads] - want) <= bound).all(), (b, t, h, (np.abs(got[b, t, heads] - want) / bound).max())
