"""GPU: the block operators (include/gpann_blocks.h) against their definitions in binary64 (tests/blocks_ref.py; the bounds are derived there)."""
import numpy as np
import pytest
import torch

import blocks_ref as ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
SENTINEL = 776.0      # a number of every type here


@pytest.fixture(scope="module")
def blocks(gp):
    from pygpann import blocks
    return blocks


class Problem:
    """random tensors of one layout, on the device and in binary64; unused places hold NaN"""

    def __init__(self, blocks, seed=0, batch=2, q_rows=5, kv_rows=150, q_heads=4, kv_heads=2, dim=64, bs=32, nprobe=4, dtype="bf16", causal=True, paged=False,
                 q_len=None, kv_len=None, packed=False, scale=None, probes=None, strength=1.0, device=0):
        self.__dict__.update(blocks=blocks, batch=batch, q_rows=q_rows, kv_rows=kv_rows, q_heads=q_heads, kv_heads=kv_heads, dim=dim, bs=bs, nprobe=nprobe,
                             dtype=dtype, causal=causal, paged=paged, G=q_heads // kv_heads, nblk=-(-kv_rows // bs), device=device)
        self.scale = dim ** -0.5 if scale is None else scale
        rng = np.random.default_rng(seed)
        dt, dev = DT[dtype], torch.device("cuda", device)
        self.kv = [kv_rows] * batch if kv_len is None else list(kv_len)
        self.ql = [q_rows] * batch if q_len is None else list(q_len)
        n_eff, m_eff = [min(max(x, 0), kv_rows) for x in self.kv], [min(max(x, 0), q_rows) for x in self.ql]
        self.n, self.m = n_eff, m_eff
        rnd = lambda *s: torch.from_numpy(rng.normal(size=s) * strength).to(dt)
        q, k, v = rnd(batch, q_rows, q_heads, dim), rnd(batch, kv_rows, kv_heads, dim), rnd(batch, kv_rows, kv_heads, dim)
        self.dout_cpu = rnd(batch, q_rows, q_heads, dim)
        self.q64, self.k64, self.v64, self.do64 = (x.double().numpy() for x in (q, k, v, self.dout_cpu))
        for b in range(batch):
            q[b, m_eff[b]:] = float("nan")
            k[b, n_eff[b]:] = float("nan")
            v[b, n_eff[b]:] = float("nan")
        if probes is None:
            probes = rng.integers(-1, self.nblk + 1, size=(batch, q_rows, kv_heads, nprobe))
        self.probes_np = np.asarray(probes, np.int32)
        self.probes = torch.from_numpy(self.probes_np).to(dev)
        extra = {}
        self.table = None
        if paged:
            self.n_pages = batch * self.nblk + 3
            table = rng.permutation(self.n_pages)[:batch * self.nblk].reshape(batch, self.nblk).astype(np.int32)
            pools = []
            for x in (k, v):
                pool = torch.full((self.n_pages, bs, kv_heads, dim), float("nan"), dtype=dt)
                for b in range(batch):
                    for j in range(self.nblk):
                        rows = x[b, j * bs:(j + 1) * bs]
                        pool[table[b, j], :rows.shape[0]] = rows
                pools.append(pool)
            k, v = pools
            self.table_np = table
            self.table = torch.from_numpy(table).to(dev)
            extra = dict(page_table=self.table.data_ptr(), n_pages=self.n_pages)
        self.q = q.to(dev)
        if packed:      # k and v are slices of one tensor
            both = torch.stack([k, v], 2).to(dev)
            self.k, self.v = both[:, :, 0], both[:, :, 1]
        else:
            self.k, self.v = k.to(dev), v.to(dev)
        self.dout = self.dout_cpu.to(dev)
        self.out = torch.full_like(self.q, SENTINEL)
        self.lse = torch.full((batch, q_rows, q_heads), SENTINEL, device=dev)
        self.kv_t = None if kv_len is None else torch.tensor(self.kv, dtype=torch.int32, device=dev)
        self.ql_t = None if q_len is None else torch.tensor(self.ql, dtype=torch.int32, device=dev)
        self.L = blocks.Layout(batch, q_rows, kv_rows, q_heads, kv_heads, dim, bs, dtype=dtype, causal=causal, scale=self.scale, device=device,
                               q_len=None if self.ql_t is None else self.ql_t.data_ptr(), kv_len=None if self.kv_t is None else self.kv_t.data_ptr(),
                               k_stride=self.k.stride()[:3], v_stride=self.v.stride()[:3], **extra)
        self.ws = torch.empty(max(16, blocks.workspace_bytes(self.L, nprobe, list(blocks.CALLS))), dtype=torch.uint8, device=dev)
        self.space = dict(workspace=self.ws.data_ptr(), workspace_bytes=self.ws.numel())

    def attend(self, stream=None):
        self.blocks.attend(self.L, self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.probes.data_ptr(), self.nprobe, self.out.data_ptr(),
                           self.lse.data_ptr(), stream=stream, **self.space)

    def rows(self):
        """(sequence, query row, key/value head, slice of query heads, rows it sees)"""
        for b in range(self.batch):
            for t in range(self.m[b]):
                for h in range(self.kv_heads):
                    yield b, t, h, slice(h * self.G, (h + 1) * self.G), ref.visible(self.n[b], self.m[b], t, self.causal)

    def pages_of(self, b):
        return None if not self.paged else [0 <= p < self.n_pages for p in self.table_np[b]]

    def check_attend(self):
        out, lse = self.out.double().cpu().numpy(), self.lse.double().cpu().numpy()
        for b, t, h, heads, vis in self.rows():
            want, want_lse, tol, tol_lse = ref.attend(self.q64[b, t, heads], self.k64[b, :, h], self.v64[b, :, h], self.probes_np[b, t, h], self.bs, self.nblk, vis,
                                                      self.scale, self.dtype, self.pages_of(b))
            assert (np.abs(out[b, t, heads] - want) <= tol).all(), (b, t, h, np.abs(out[b, t, heads] - want).max(), tol.max())
            got = lse[b, t, heads]
            empty = np.isinf(want_lse)
            assert np.array_equal(got == -np.inf, empty) and (np.abs(got - want_lse)[~empty] <= tol_lse[~empty]).all(), (b, t, h, got, want_lse)
        for b in range(self.batch):      # rows behind the last of a sequence are left alone
            assert (out[b, self.m[b]:] == SENTINEL).all() and (lse[b, self.m[b]:] == SENTINEL).all()

    def backward(self, stream=None):
        self.dq = torch.full_like(self.q, float("nan"))
        self.dk, self.dv = (torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=x.device) for x in (self.k, self.v))
        self.dk.fill_(float("nan"))
        self.dv.fill_(float("nan"))
        self.backward_call(stream)

    def backward_call(self, stream=None):
        p = lambda x: x.data_ptr()
        self.blocks.attend_backward(self.L, p(self.q), p(self.k), p(self.v), p(self.probes), self.nprobe, p(self.out), p(self.lse), p(self.dout), p(self.dq), p(self.dk),
                                    p(self.dv), stream=stream, **self.space)

    def check_backward(self):
        u = ref.U[self.dtype]
        got = {x: getattr(self, x).double().cpu().numpy() for x in ("dq", "dk", "dv")}
        want = {x: np.zeros(y.shape) for x, y in got.items()}
        tol = {x: np.zeros(y.shape) for x, y in got.items()}
        terms = np.zeros(self.k64.shape[:3])
        size = {x: np.zeros(got[x].shape) for x in ("dk", "dv")}
        for b, t, h, heads, vis in self.rows():
            rows, dq, dk, dv, eq, ek, ev = ref.backward(self.q64[b, t, heads], self.k64[b, :, h], self.v64[b, :, h], self.do64[b, t, heads],
                                                        self.probes_np[b, t, h], self.bs, self.nblk, vis, self.scale, self.dtype)
            want["dq"][b, t, heads], tol["dq"][b, t, heads] = dq, eq
            if len(rows):
                for x, y, e in (("dk", dk, ek), ("dv", dv, ev)):
                    want[x][b, rows, h] += y
                    tol[x][b, rows, h] += e
                    size[x][b, rows, h] += np.abs(y) + e
                terms[b, rows, h] += self.G
        for x in ("dk", "dv"):           # the sums over query rows and heads are in binary32
            tol[x] += (terms[..., None] + 8) * ref.E * size[x]
        tiny = 2.0 ** -24 if self.dtype == "fp16" else 0.0      # half a step of the type's smallest numbers
        for x in got:
            bound = tol[x] + u * (np.abs(want[x]) + tol[x]) + tiny
            bad = ~(np.abs(got[x] - want[x]) <= bound)
            assert not bad.any(), (x, np.argwhere(bad)[:4], np.abs(got[x] - want[x])[bad][:4], bound[bad][:4])


SHAPES = [
    dict(dim=64), dict(dim=96, dtype="fp16"), dict(dim=128), dict(dim=192, dtype="fp16"), dict(dim=256), dict(dim=256, dtype="fp16", bs=16),
    dict(q_heads=2, kv_heads=2, bs=16), dict(q_heads=6, kv_heads=2, bs=48, kv_rows=301), dict(q_heads=5, kv_heads=1, bs=64), dict(q_heads=8, kv_heads=1, bs=256, kv_rows=700),
    dict(q_heads=32, kv_heads=2, bs=16, dim=128), dict(q_heads=20, kv_heads=1), dict(q_heads=40, kv_heads=1, dim=96, q_rows=3), dict(causal=False, q_rows=7),
    dict(packed=True), dict(batch=1, q_rows=1, q_heads=1, kv_heads=1, kv_rows=1, nprobe=1), dict(batch=1, q_rows=1, kv_rows=4000, bs=64, nprobe=64, dim=128),
    dict(q_rows=70, kv_rows=70, bs=16, nprobe=3), dict(q_rows=131, kv_rows=257, bs=32, nprobe=9, batch=1), dict(nprobe=33, kv_rows=1100),
    dict(q_len=[5, 0], kv_len=[150, 150]), dict(q_len=[3, 5], kv_len=[1, 31]), dict(q_len=[5, 4], kv_len=[0, 3]), dict(q_len=[99, -3], kv_len=[999, 20]),
    dict(q_len=[5, 4], kv_len=[0, 3], causal=False), dict(strength=3.0), dict(scale=-0.2), dict(scale=0.0), dict(batch=3, q_rows=33, kv_rows=97, kv_heads=1, q_heads=16),
    dict(q_rows=1, q_heads=24, kv_heads=8, batch=5, kv_len=[150, 7, 64, 65, 1]),
    dict(batch=1, q_rows=1300, kv_rows=1300, q_heads=16, kv_heads=1, bs=64, nprobe=3),            # blocks that more rows probe than one workgroup takes
    dict(batch=1, q_rows=1100, kv_rows=1200, q_heads=32, kv_heads=1, bs=16, nprobe=3, dtype="fp16"), dict(batch=1, q_rows=300, kv_rows=300, q_heads=24, kv_heads=1, bs=128, dim=192),
    dict(batch=1, q_rows=20, kv_rows=20000, bs=16, nprobe=40, q_heads=3, kv_heads=1),             # more blocks than a walk holds at a time
    dict(batch=1, q_rows=4, kv_rows=18000, bs=16, nprobe=64, q_heads=2, kv_heads=1, dim=192), dict(q_rows=260, kv_rows=260, q_heads=2, kv_heads=2, bs=96, batch=1),
    dict(batch=8, q_rows=96, kv_rows=128, q_heads=64, kv_heads=8, dim=128, bs=32), dict(batch=8, q_rows=250, kv_rows=256, q_heads=24, kv_heads=8, dim=64, bs=16, causal=False),
]


@pytest.mark.parametrize("kw", SHAPES, ids=lambda x: "-".join(f"{k}{v}" for k, v in x.items()))
def test_attend(blocks, kw):
    p = Problem(blocks, seed=11, **kw)
    p.attend()
    torch.cuda.synchronize()
    p.check_attend()


@pytest.mark.parametrize("kw", SHAPES, ids=lambda x: "-".join(f"{k}{v}" for k, v in x.items()))
def test_backward(blocks, kw):
    p = Problem(blocks, seed=12, **kw)
    p.attend()
    p.backward()
    torch.cuda.synchronize()
    p.check_backward()
    first = [x.clone() for x in (p.dq, p.dk, p.dv)]
    p.backward()      # every sum has one order
    for x, y in zip(first, (p.dq, p.dk, p.dv)):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("kw", [dict(), dict(bs=64, dim=128, q_rows=1, batch=3), dict(bs=16, dtype="fp16", q_heads=16, kv_heads=1), dict(q_rows=40, kv_len=[150, 33], q_len=[40, 2])],
                         ids=str)
def test_attend_paged(blocks, kw):
    p = Problem(blocks, seed=13, paged=True, **kw)
    p.attend()
    torch.cuda.synchronize()
    p.check_attend()


WALKS = [
    dict(), dict(dim=96, bs=48, dtype="fp16"), dict(dim=128, bs=64), dict(dim=192, bs=16, dtype="fp16"), dict(dim=256, bs=128), dict(q_heads=8, bs=16, dim=128),
    dict(q_heads=24, bs=64, dtype="fp16"), dict(q_heads=80, kv_heads=4, q_rows=70), dict(q_heads=128, bs=64), dict(causal=False, bs=256, kv_rows=600), dict(scale=-0.2), dict(scale=0.0),
    dict(packed=True), dict(kv_len=[0, 1, 33, 150, 149, 64, 16, 97], q_len=[40, 40, 3, 40, 0, 17, 40, 33]), dict(paged=True, bs=16, nprobe=9), dict(paged=True, bs=64, dim=128, kv_rows=301),
    dict(batch=1, kv_heads=1, q_heads=2, q_rows=2100, kv_rows=20000, bs=16, nprobe=5), dict(batch=1, kv_heads=1, q_heads=2, q_rows=2100, kv_rows=9000, bs=16, nprobe=5, dim=128),
    dict(batch=3, kv_heads=4, q_heads=12, q_rows=300, kv_rows=700, dim=96, dtype="fp16", nprobe=12), dict(batch=16, q_heads=32, q_rows=129, dim=128, bs=64, kv_rows=256),
    # enough of them for 32 columns a wavefront
    *(dict(batch=16, kv_heads=16, q_heads=256, q_rows=20, **kw) for kw in (dict(bs=16), dict(dim=96, dtype="fp16"), dict(dim=128, bs=64), dict(dim=128, bs=48, dtype="fp16", causal=False))),
    dict(batch=16, kv_heads=16, q_heads=640, q_rows=8, bs=64), dict(batch=16, kv_heads=16, q_heads=48, q_rows=90, bs=64, q_len=[90, 3] * 8, kv_len=[150, 149, 64, 65, 1, 0, 33, 96] * 2),
]


@pytest.mark.parametrize("kw", WALKS, ids=lambda x: "-".join(f"{k}{v}" for k, v in x.items()))
def test_attend_many_rows_together(blocks, kw):
    """more wavefronts of query rows than the chip has: neighbours walk the blocks that any of them probes"""
    p = Problem(blocks, **{**dict(seed=71, batch=8, q_rows=40, q_heads=16, kv_heads=8), **kw})
    p.attend()
    torch.cuda.synchronize()
    p.check_attend()


@pytest.mark.parametrize("kw", [dict(batch=1, q_heads=128, kv_heads=64), dict(batch=8, q_heads=128, kv_heads=64), dict(batch=32, q_heads=640, kv_heads=16), dict(batch=16, dim=128)], ids=str)
def test_many_rows_beside_values_that_are_not_numbers(blocks, kw):
    """as above, with 16 and 32 columns a wavefront"""
    kw = {**dict(batch=1, q_heads=512, kv_heads=32), **kw}
    probes = np.full((kw["batch"], 40, kw["kv_heads"], 3), -1, np.int32)
    probes[:, :, :, 0] = 0
    probes[:, ::2, :, 1] = 1            # every second row looks at block 1, which holds the values that are none
    probes[:, :, :, 2] = 4
    p = Problem(blocks, seed=72, q_rows=40, kv_rows=150, probes=probes, nprobe=3, **kw)
    p.v[:, 40], p.v[:, 41], p.k[:, 42], p.v[:, 140] = float("inf"), float("nan"), float("nan"), float("inf")   # row 140: seen by the rows from t = 30 on
    p.attend()
    torch.cuda.synchronize()
    out = p.out.double().cpu().numpy()
    for b, t, h, heads, vis in p.rows():
        if b not in (0, p.batch - 1) or h % 5:
            continue
        want, _, tol, _ = ref.attend(p.q64[b, t, heads], p.k64[b, :, h], p.v64[b, :, h], probes[b, t, h], p.bs, p.nblk, vis, p.scale, p.dtype)
        if t % 2 == 0:
            assert np.isnan(out[b, t, heads]).all()
        elif vis > 140:
            assert (out[b, t, heads] == np.inf).all()
        else:
            assert (np.abs(out[b, t, heads] - want) <= tol).all()


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("kw", [dict(bs=16, q_heads=6), dict(bs=48, q_heads=2, dtype="fp16"), dict(bs=64, q_heads=80, paged=True), dict(bs=256, q_heads=34, dtype="fp16", causal=False)], ids=str)
def test_single_tokens_at_every_length(blocks, dim, kw):
    """one query row a sequence: lengths around the tiles, keys divided over workgroups, pages that end inside a tile, an infinity in the last row"""
    lens = [0, 1, 15, 16, 17, 47, 49, 700]
    probes = np.random.default_rng(3).permuted(np.tile(np.arange(44), (8, 1, 2, 1)), axis=-1)[..., :40]
    probes[..., 0] = 0
    p = Problem(blocks, seed=19, batch=8, q_rows=1, kv_rows=700, kv_heads=2, dim=dim, kv_len=lens, nprobe=40, probes=probes, **kw)
    p.attend()
    torch.cuda.synchronize()
    p.check_attend()
    if not p.paged:
        p.v[1, 0, :, 3], p.v[6, 48, :, 5] = float("inf"), float("inf")      # seen by one sequence's token: its weight is not 0
        p.attend()
        torch.cuda.synchronize()
        assert (p.out[1, 0, :, 3] == float("inf")).all() and torch.isfinite(p.out[1, 0, :, 4:]).all()
        seen = torch.from_numpy((p.probes_np[6, 0] == 48 // p.bs).any(-1)).repeat_interleave(p.G).cuda()
        assert torch.equal(p.out[6, 0, :, 5] == float("inf"), seen) and torch.isfinite(p.out[6, 0, :, 6:]).all()


def test_pages_that_do_not_exist_are_skipped(blocks):
    p = Problem(blocks, seed=14, paged=True)
    p.table_np[0, 1], p.table_np[1, 2], p.table_np[0, 3] = -1, p.n_pages, -2 ** 31
    p.table.copy_(torch.from_numpy(p.table_np))
    p.attend()
    torch.cuda.synchronize()
    p.check_attend()


def test_probe_rows_with_repeats_strays_and_nothing(blocks):
    probes = np.tile(np.array([[2, 2, 0, 2], [-1, -1, -1, -1], [4, 99, -7, 4], [2 ** 31 - 1, -2 ** 31, 1, 0], [3, 2, 1, 0]], np.int32)[None, :, None, :], (2, 1, 2, 1))
    for causal in (True, False):
        p = Problem(blocks, seed=15, probes=probes, causal=causal)
        p.attend()
        p.backward()
        torch.cuda.synchronize()
        p.check_attend()
        p.check_backward()
        assert (p.out[:, 1] == 0).all() and torch.isinf(p.lse[:, 1]).all()


def test_values_that_are_not_numbers_reach_only_the_rows_that_see_them(blocks):
    """a NaN and infinities in keys and values of rows that other query rows of the same call do not look at"""
    probes = np.full((1, 40, 2, 3), -1, np.int32)
    probes[0, :, :, 0] = 0
    probes[0, ::2, :, 1] = 1            # every second row looks at block 1, which holds the values that are none
    probes[0, :, :, 2] = 4
    p = Problem(blocks, seed=16, batch=1, q_rows=40, kv_rows=150, probes=probes, nprobe=3)
    p.v[0, 40], p.v[0, 41], p.k[0, 42], p.v[0, 140] = float("inf"), float("nan"), float("nan"), float("inf")   # row 140: seen by the rows from t = 30 on
    p.attend()
    torch.cuda.synchronize()
    out = p.out.double().cpu().numpy()
    for b, t, h, heads, vis in p.rows():
        want, _, tol, _ = ref.attend(p.q64[b, t, heads], p.k64[b, :, h], p.v64[b, :, h], probes[b, t, h], p.bs, p.nblk, vis, p.scale, p.dtype)
        if t % 2 == 0:
            assert np.isnan(out[b, t, heads]).all()
        elif vis > 140:
            assert (out[b, t, heads] == np.inf).all()
        else:
            assert (np.abs(out[b, t, heads] - want) <= tol).all()


@pytest.mark.parametrize("kw", [dict(), dict(dim=128, bs=64, kv_rows=400), dict(dim=192, dtype="fp16"), dict(dim=256, bs=16, kv_rows=100)], ids=str)
def test_gradients_of_rows_that_do_not_see_what_is_not_a_number(blocks, kw):
    """odd query rows look at blocks 0 and 4, even ones at blocks 1 and 2, which hold a NaN and infinities"""
    probes = np.full((1, 40, 2, 3), -1, np.int32)
    probes[0, 1::2, :, :2], probes[0, ::2, :, :2] = (0, 4), (1, 2)
    p = Problem(blocks, **{**dict(seed=18, batch=1, q_rows=40, kv_rows=200, probes=probes, nprobe=3), **kw})
    bs = p.bs
    p.v[0, bs + 1], p.v[0, bs + 2], p.k[0, 2 * bs + 3] = float("inf"), float("nan"), float("nan")
    p.attend()
    p.backward()
    torch.cuda.synchronize()
    assert torch.isnan(p.dq[0, ::2]).all()
    p.dq[0, ::2] = 0
    for x in (p.dk, p.dv):
        x[0, bs:3 * bs] = 0
    every = p.rows
    p.rows = lambda: (row for row in every() if row[1] % 2)
    p.check_backward()


def test_blocks_that_lie_beyond_32_bits(blocks):
    """pages 2^31 elements apart"""
    p = Problem(blocks, seed=17, batch=1, kv_rows=96, paged=True, nprobe=3)
    far = 2 ** 30
    for name in ("k", "v"):
        x = getattr(p, name)
        big = torch.empty(far * (x.shape[0] - 1) + x[0].numel(), dtype=x.dtype, device="cuda")
        view = torch.as_strided(big, x.shape, (far, *x.stride()[1:]))
        view.copy_(x)
        setattr(p, name, view)
    p.L = blocks.Layout(1, p.q_rows, 96, 4, 2, 64, 32, kv_len=None, page_table=p.table.data_ptr(), n_pages=p.n_pages, k_stride=p.k.stride()[:3], v_stride=p.v.stride()[:3])
    p.attend()
    torch.cuda.synchronize()
    p.check_attend()


# ---- routing ----------------------------------------------------------------------------------------------------------------------------------
def _summaries(p):
    s = torch.full((p.batch, p.kv_heads, p.nblk, p.dim), SENTINEL, device="cuda")
    p.blocks.summarize(p.L, p.k.data_ptr(), s.data_ptr())
    return s


@pytest.mark.parametrize("kw", [dict(), dict(dim=96, bs=48), dict(dim=256, bs=16, dtype="fp16"), dict(kv_len=[0, 150]), dict(kv_len=[1, 33], dim=192), dict(paged=True, dim=128),
                                dict(packed=True), dict(bs=256, kv_rows=600)], ids=str)
def test_summaries(blocks, kw):
    p = Problem(blocks, seed=21, **kw)
    s = _summaries(p).cpu().numpy()
    for b in range(p.batch):
        nb = -(-p.n[b] // p.bs)
        for h in range(p.kv_heads):
            assert np.array_equal(s[b, h, :nb], ref.summarize(p.k64[b, :, h], p.n[b], p.bs))
        assert (s[b, :, nb:] == SENTINEL).all()


@pytest.mark.parametrize("new_rows", [1, 2, 31, 32, 33, 40, 10 ** 6])
def test_summaries_of_the_new_rows_only(blocks, new_rows):
    p = Problem(blocks, seed=22, kv_len=[150, 65])
    want = _summaries(p).cpu()
    s = torch.full_like(want, SENTINEL).cuda()
    blocks.summarize(p.L, p.k.data_ptr(), s.data_ptr(), new_rows=new_rows)
    s = s.cpu()
    for b in range(2):
        first = max(0, p.n[b] - new_rows) // p.bs
        assert torch.equal(s[b, :, first:], want[b, :, first:]) and (s[b, :, :first] == SENTINEL).all()


ROUTES = [dict(), dict(nprobe=3), dict(nprobe=1, first=0, last=1), dict(kv_rows=3000, bs=16, nprobe=40, q_rows=3), dict(kv_rows=5000, bs=16, nprobe=64, q_rows=2, q_heads=16, kv_heads=1),
          dict(causal=False, nprobe=3, first=0, last=0), dict(q_heads=2, kv_heads=2, dim=96, nprobe=3), dict(dim=256, dtype="fp16", nprobe=3), dict(q_len=[5, 0], kv_len=[0, 40]),
          dict(q_len=[2, 5], kv_len=[150, 3], nprobe=3), dict(paged=True, nprobe=3, dim=192), dict(q_rows=150, nprobe=3, batch=1), dict(q_rows=300, kv_rows=1999, nprobe=7, batch=1, dim=128),
          dict(q_rows=70, kv_rows=4100, bs=32, nprobe=16, batch=2, dim=64, q_len=[70, 33], kv_len=[4100, 3333])]


@pytest.mark.parametrize("kw", ROUTES, ids=str)
def test_route(blocks, kw):
    kw = dict(kw)
    first, last = kw.pop("first", 1), kw.pop("last", 2)
    p = Problem(blocks, seed=23, **kw)
    s = _summaries(p)
    probes = torch.full_like(p.probes, 12345)
    blocks.route(p.L, p.q.data_ptr(), s.data_ptr(), p.nprobe, probes.data_ptr(), first=first, last=last, **p.space)
    got, cen = probes.cpu().numpy(), s.cpu().numpy()
    for b, t, h, heads, vis in p.rows():
        assert np.array_equal(got[b, t, h], ref.route(p.q64[b, t, heads], cen[b, h], p.bs, vis, p.nprobe, first, last)), (b, t, h)
    for b in range(p.batch):
        assert (got[b, p.m[b]:] == 12345).all()


@pytest.mark.parametrize("kw", [dict(dim=96, dtype="fp16"), dict(dim=192, q_heads=8), dict(dim=256, bs=16, q_heads=128), dict(dim=128, q_rows=23, kv_len=[150, 149, 1, 0], q_len=[23, 2, 23, 1]),
                                dict(kv_rows=9000, bs=16, nprobe=30, q_rows=17), dict(kv_rows=5000, bs=16, nprobe=64, causal=False), dict(paged=True, dim=128, nprobe=5), dict(scale=-1.0)], ids=str)
def test_route_by_tiles_of_query_rows(blocks, kw):
    test_route(blocks, {**dict(batch=4, kv_heads=8, q_heads=16, q_rows=9, nprobe=3), **kw})


def test_route_ties_and_values_that_are_not_numbers(blocks):
    p = Problem(blocks, seed=24, batch=1, kv_rows=640, bs=16, nprobe=6, q_rows=20)
    s = _summaries(p)
    s[0, 0] = s[0, 0, 7].clone()                    # all blocks score the same: the lowest are taken
    s[0, 1, 3:30:2] = s[0, 1, 3].clone()
    s[0, 1, 5], s[0, 1, 10] = float("nan"), float("inf")
    s[0, 1, 12] = -0.0 * s[0, 1, 12]
    probes = torch.empty_like(p.probes)
    blocks.route(p.L, p.q.data_ptr(), s.data_ptr(), p.nprobe, probes.data_ptr(), first=0, last=1, **p.space)
    got, cen = probes.cpu().numpy(), s.cpu().numpy()
    with np.errstate(invalid="ignore"):
        for b, t, h, heads, vis in p.rows():
            assert np.array_equal(got[b, t, h], ref.route(p.q64[b, t, heads], cen[b, h], p.bs, vis, p.nprobe, 0, 1)), (t, h)
    s.fill_(float("nan"))
    blocks.route(p.L, p.q.data_ptr(), s.data_ptr(), p.nprobe, probes.data_ptr(), first=0, last=1, **p.space)
    for b, t, h, heads, vis in p.rows():
        nb = -(-vis // p.bs)
        assert list(probes[b, t, h].cpu().numpy()) == [0, 1, 2, 3, 4, nb - 1]


# ---- weights and eviction ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(q_rows=1), dict(q_rows=1, q_heads=40, kv_heads=1), dict(q_rows=1, kv_len=[0, 77]), dict(q_rows=1, paged=True, bs=16, dim=128), dict(), dict(paged=True),
                                dict(q_rows=40, bs=256, kv_rows=600, dim=256), dict(q_rows=3, q_heads=20, kv_heads=1, bs=16, dtype="fp16"), dict(q_len=[5, 0], kv_len=[3, 150]),
                                dict(causal=False, dim=96), dict(q_rows=1, causal=False, dim=192, bs=48)], ids=str)
@pytest.mark.parametrize("in_place", [False, True])
def test_weigh(blocks, kw, in_place):
    p = Problem(blocks, seed=31, **kw)
    p.attend()
    mass = torch.rand(p.batch, p.kv_heads, p.kv_rows, device="cuda")
    before = mass.double().cpu().numpy()
    out = mass if in_place else torch.full_like(mass, SENTINEL)
    blocks.weigh(p.L, p.q.data_ptr(), p.k.data_ptr(), p.probes.data_ptr(), p.nprobe, p.lse.data_ptr(), mass.data_ptr(), out.data_ptr(), **p.space)
    got = out.double().cpu().numpy()
    want, tol, touched = before.copy(), np.zeros_like(before), np.zeros(before.shape, bool)
    for b, t, h, heads, vis in p.rows():
        rows = ref.rows_of(p.probes_np[b, t, h], p.bs, p.nblk, vis)
        if len(rows):
            lse, pr, w = ref.softmax_rows(p.q64[b, t, heads], p.k64[b, rows, h], p.scale)
            want[b, h, rows] += pr.sum(0)
            touched[b, h, rows] = True
            tol[b, h, rows] += (pr * (3 * w + 4 * ref.E * np.abs(lse).max())).sum(0)
    tol += ref.E * (p.G * p.q_rows + 4) * want        # binary32 sums
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    assert np.array_equal(got[~touched], before[~touched])


@pytest.mark.parametrize("kw", [dict(kv_rows=1000, kv_len=[1000, 700]), dict(kv_rows=1001, kv_len=[999, 1001], nprobe=20, dtype="fp16", dim=96), dict(kv_rows=3000, bs=256, paged=True)],
                         ids=str)
@pytest.mark.parametrize("in_place", [False, True])
def test_weigh_a_token_divided_over_workgroups(blocks, kw, in_place):
    test_weigh(blocks, {**dict(q_rows=1, bs=128, nprobe=7), **kw}, in_place)


@pytest.mark.parametrize("kw", [dict(keep=50), dict(keep=50, first=4, last=10), dict(keep=1), dict(keep=150), dict(keep=400), dict(keep=149, last=1), dict(keep=7, first=3, last=4),
                                dict(keep=60, kv_len=[0, 61]), dict(keep=33, paged=True, bs=16, first=1), dict(keep=40, ties=True), dict(keep=40, ties=True, kv_rows=3000, last=5),
                                dict(keep=2000, kv_rows=5000, dim=256, dtype="fp16", kv_heads=1), dict(keep=900, kv_rows=1024, packed=True)], ids=str)
def test_evict(blocks, kw):
    kw = dict(kw)
    keep, first, last, ties = kw.pop("keep"), kw.pop("first", 0), kw.pop("last", 0), kw.pop("ties", False)
    p = Problem(blocks, seed=41, **kw)
    rng = np.random.default_rng(1)
    mass = rng.random((p.batch, p.kv_heads, p.kv_rows)).astype(np.float32)
    if ties:
        mass = (mass * 3).astype(np.int32).astype(np.float32) - 1
        mass[0, 0, 10:20], mass[0, 0, 30] = np.nan, -0.0
    m = torch.from_numpy(mass).cuda()
    rows = torch.full((p.batch, p.kv_heads, keep), -5, dtype=torch.int32, device="cuda")
    count = torch.full((p.batch, p.kv_heads), -5, dtype=torch.int32, device="cuda")
    k_out, v_out = (torch.full((p.batch, keep, p.kv_heads, p.dim), SENTINEL, dtype=DT[p.dtype], device="cuda") for _ in range(2))
    mass_out = torch.full((p.batch, p.kv_heads, keep), SENTINEL, device="cuda")
    blocks.evict(p.L, p.k.data_ptr(), p.v.data_ptr(), m.data_ptr(), keep, rows.data_ptr(), count.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), mass_out.data_ptr(),
                 first=first, last=last, **p.space)
    for b in range(p.batch):
        for h in range(p.kv_heads):
            want = ref.evict(mass[b, h], p.n[b], keep, first, last)
            c = len(want)
            assert count[b, h] == c and rows[b, h, :c].tolist() == want, (b, h)
            assert (rows[b, h, c:] == -5).all() and (k_out[b, c:, h] == SENTINEL).all() and (v_out[b, c:, h] == SENTINEL).all() and (mass_out[b, h, c:] == SENTINEL).all()
            if c:
                assert np.array_equal(k_out[b, :c, h].double().cpu().numpy(), p.k64[b, want, h]) and np.array_equal(v_out[b, :c, h].double().cpu().numpy(), p.v64[b, want, h])
                assert np.array_equal(mass_out[b, h, :c].cpu().numpy(), mass[b, h, want], equal_nan=True)
    again = torch.full_like(rows, -5)
    blocks.evict(p.L, None, None, m.data_ptr(), keep, again.data_ptr(), count.data_ptr(), first=first, last=last, **p.space)     # selection alone
    assert torch.equal(again, rows)


# ---- streams, graphs, a run of them together ----------------------------------------------------------------------------------------------------
def test_calls_on_another_stream_and_two_at_once(blocks):
    a, b = Problem(blocks, seed=51, q_rows=60, kv_rows=400), Problem(blocks, seed=52, q_rows=60, kv_rows=400)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        for p, st in ((a, s), (b, t)):
            p.attend(stream=st.cuda_stream)
    s.synchronize()
    t.synchronize()
    with torch.cuda.stream(s):
        a.backward(stream=s.cuda_stream)
    with torch.cuda.stream(t):
        b.backward(stream=t.cuda_stream)
    torch.cuda.synchronize()
    for p in (a, b):
        p.check_attend()
        p.check_backward()


@pytest.mark.parametrize("kw", [dict(q_rows=1, kv_rows=1000, bs=64), dict(q_rows=33, kv_rows=300)], ids=str)
def test_a_captured_step_replays(blocks, kw):
    """route, attend, weigh, evict (and the gradients) captured once and replayed on new inputs, with eager calls between the replays"""
    p, other = Problem(blocks, seed=53, **kw), Problem(blocks, seed=54, **kw)
    s = _summaries(p)
    mass, mass_out = torch.zeros(p.batch, p.kv_heads, p.kv_rows, device="cuda"), torch.empty(p.batch, p.kv_heads, p.kv_rows, device="cuda")
    keep = 40
    rows, count = torch.zeros(p.batch, p.kv_heads, keep, dtype=torch.int32, device="cuda"), torch.zeros(p.batch, p.kv_heads, dtype=torch.int32, device="cuda")
    k_out, v_out = (torch.zeros(p.batch, keep, p.kv_heads, p.dim, dtype=DT[p.dtype], device="cuda") for _ in range(2))
    p.dq, p.dk, p.dv = torch.zeros_like(p.q), torch.zeros_like(p.k), torch.zeros_like(p.v)
    outs = (p.probes, p.out, p.lse, mass_out, rows, count, k_out, v_out, p.dq, p.dk, p.dv)

    def step(stream):
        blocks.summarize(p.L, p.k.data_ptr(), s.data_ptr(), new_rows=p.q_rows, stream=stream)
        blocks.route(p.L, p.q.data_ptr(), s.data_ptr(), p.nprobe, p.probes.data_ptr(), stream=stream, **p.space)
        p.attend(stream)
        blocks.weigh(p.L, p.q.data_ptr(), p.k.data_ptr(), p.probes.data_ptr(), p.nprobe, p.lse.data_ptr(), mass.data_ptr(), mass_out.data_ptr(), stream=stream, **p.space)
        blocks.evict(p.L, p.k.data_ptr(), p.v.data_ptr(), mass_out.data_ptr(), keep, rows.data_ptr(), count.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), first=1, last=4,
                     stream=stream, **p.space)
        p.backward_call(stream)

    step(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for i in range(3):
        p.q.copy_(other.q * (1 + i))
        p.v.copy_(other.v)
        mass.fill_(0.25 * i)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs]
        other.attend()                                  # eager work between the replays
        step(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for x, y in zip(got, outs):
            assert torch.equal(x, y)


def test_a_cache_is_used_as_a_serving_program_uses_it(blocks):
    """prompt -> routed attention, weights, eviction, then tokens attend to what was kept: every step against the definitions"""
    p = Problem(blocks, seed=55, batch=2, q_rows=64, kv_rows=512, q_heads=8, kv_heads=2, dim=128, bs=32, nprobe=6, kv_len=[512, 300], q_len=[64, 20])
    s = _summaries(p)
    blocks.route(p.L, p.q.data_ptr(), s.data_ptr(), p.nprobe, p.probes.data_ptr(), first=1, last=2, **p.space)
    p.probes_np = p.probes.cpu().numpy()
    p.attend()
    p.check_attend()
    mass = torch.zeros(2, 2, 512, device="cuda")
    blocks.weigh(p.L, p.q.data_ptr(), p.k.data_ptr(), p.probes.data_ptr(), p.nprobe, p.lse.data_ptr(), mass.data_ptr(), mass.data_ptr(), **p.space)
    total = mass.sum(2).cpu()                           # every (query row, head) spreads a weight of 1
    for b in range(2):
        assert torch.allclose(total[b], torch.full((2,), 4.0 * p.m[b]), rtol=1e-4)
    keep = 128
    rows, count = torch.zeros(2, 2, keep, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    k_out, v_out = (torch.zeros(2, keep, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    blocks.evict(p.L, p.k.data_ptr(), p.v.data_ptr(), mass.data_ptr(), keep, rows.data_ptr(), count.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), first=4, last=32, **p.space)
    kept, weights = rows.cpu().numpy(), mass.cpu().numpy()
    for b in range(2):
        for h in range(2):
            assert kept[b, h].tolist() == ref.evict(weights[b, h], p.n[b], keep, 4, 32)
    t = Problem(blocks, seed=56, batch=2, q_rows=1, kv_rows=keep, q_heads=8, kv_heads=2, dim=128, bs=32, nprobe=4, probes=np.tile(np.arange(4, dtype=np.int32), (2, 1, 2, 1)))
    t.k, t.v = k_out, v_out
    t.k64, t.v64 = k_out.double().cpu().numpy(), v_out.double().cpu().numpy()
    t.attend()
    t.check_attend()


def test_the_current_device_and_another_devices_stream(blocks):
    p = Problem(blocks, seed=57)
    p.attend()
    assert torch.cuda.current_device() == 0
    p.check_attend()
    L = blocks.Layout(1, 1, 64, 1, 1, 64, 32, device=99)
    with pytest.raises(blocks.GpannError):
        blocks.attend(L, 16, 16, 16, 16, 1, 16)
