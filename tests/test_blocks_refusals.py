"""CPU: the block operators' exports, layout of the argument block, refusals, and the reference's gradients against differences."""
import ctypes
import os
import re

import numpy as np
import pytest

import blocks_ref as ref
from conftest import ROOT

OK = 16   # an aligned address that is never followed: every call below is refused before anything is launched


@pytest.fixture(scope="module")
def blocks():
    import pygpann
    if not os.path.exists(pygpann.LIB_PATH):
        pygpann.build()
    from pygpann import blocks
    return blocks


def _layout(blocks, **kw):
    args = dict(batch=2, q_rows=3, kv_rows=100, q_heads=4, kv_heads=2, head_dim=64, block_rows=32)
    args.update(kw)
    return blocks.Layout(**args)


def _calls(blocks, L, **kw):
    """every entry point on this layout, with one argument replaced"""
    def use(**defaults):
        return {x: kw.get(x, y) for x, y in defaults.items()}
    ws = dict(workspace=OK, workspace_bytes=1 << 30)
    t = use(q=OK, k=OK, v=OK, probes=OK, nprobe=4)
    return {
        "summarize": lambda: blocks.summarize(L, t["k"], kw.get("summary", OK), kw.get("new_rows", 0)),
        "route": lambda: blocks.route(L, t["q"], kw.get("summary", OK), t["nprobe"], t["probes"], **use(first=1, last=2), **ws),
        "attend": lambda: blocks.attend(L, t["q"], t["k"], t["v"], t["probes"], t["nprobe"], kw.get("out", OK), kw.get("lse", OK), **ws),
        "backward": lambda: blocks.attend_backward(L, t["q"], t["k"], t["v"], t["probes"], t["nprobe"], kw.get("out", OK), kw.get("lse", OK), kw.get("dout", OK),
                                                   kw.get("dq", OK), kw.get("dk", OK), kw.get("dv", OK), **{**ws, **{x: kw[x] for x in ws if x in kw}}),
        "weigh": lambda: blocks.weigh(L, t["q"], t["k"], t["probes"], t["nprobe"], kw.get("lse", OK), kw.get("mass", OK), kw.get("mass_out", OK),
                                      **{**ws, **{x: kw[x] for x in ws if x in kw}}),
        "evict": lambda: blocks.evict(L, t["k"], t["v"], kw.get("mass", OK), kw.get("keep", 16), kw.get("rows", OK), kw.get("count", OK), kw.get("k_out", 32),
                                      kw.get("v_out", 48), kw.get("mass_out", 64), **use(first=1, last=2, out_kv_stride=None), **ws),
    }


def _refused(blocks, call, status=1, match=None):
    with pytest.raises(blocks.GpannError, match=match) as e:
        call()
    assert e.value.status == status, str(e.value)


def test_header_library_and_binding_agree(blocks):
    text = open(os.path.join(ROOT, "include", "gpann_blocks.h")).read()
    code = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = sorted(set(re.findall(r"\b(gpann_blocks_[a-z_0-9]+)\s*\(", code)))
    assert names == sorted(blocks.EXPORTS)
    L = blocks.lib()
    for n in names:
        assert hasattr(L, n)
    fields = re.search(r"typedef struct gpann_blocks_layout \{(.*?)\} gpann_blocks_layout;", code, re.S).group(1)
    declared = re.findall(r"(\w+)(?:\[3\])?\s*[,;]", fields)
    assert declared == [f for f, _ in blocks._Layout._fields_]
    assert ctypes.sizeof(blocks._Layout) == 12 * 4 + 3 * 8 + 2 * 4 + 12 * 8


@pytest.mark.parametrize("change", [
    dict(dtype=7), dict(q_heads=5), dict(q_heads=0), dict(kv_heads=0), dict(q_heads=2048, kv_heads=2), dict(head_dim=80), dict(head_dim=0), dict(head_dim=512),
    dict(block_rows=0), dict(block_rows=24), dict(block_rows=272), dict(kv_rows=16385 * 16, block_rows=16), dict(q_rows=1 << 25), dict(batch=1 << 17),
    dict(scale=float("inf")), dict(scale=float("nan")), dict(q_stride=(768, 256, 4)), dict(k_stride=(-8, 128, 64)), dict(out_stride=(1 << 41, 256, 64)),
    dict(page_table=OK, page_stride=3, n_pages=9), dict(page_table=OK, n_pages=1 << 31)])
def test_layouts_that_are_refused(blocks, change):
    def layouts():
        if "dtype" in change:
            L = _layout(blocks)
            L.c.dtype = change["dtype"]
            return L
        return _layout(blocks, **change)
    L = layouts()
    for name, call in _calls(blocks, L).items():
        _refused(blocks, call)
    _refused(blocks, lambda: blocks.workspace_bytes(L, 4, ["backward"]))


def test_unknown_flags_and_struct_sizes_are_refused(blocks):
    L = _layout(blocks)
    L.c.flags |= 2
    _refused(blocks, _calls(blocks, L)["attend"], match="flags")
    L = _layout(blocks)
    L.c.struct_bytes -= 8
    _refused(blocks, _calls(blocks, L)["attend"], match="struct_bytes")
    assert blocks.lib().gpann_blocks_attend(None, None, None, None, None, 1, None, None, None, 0, None) == 1
    with pytest.raises(blocks.GpannError):
        blocks.Layout(1, 1, 64, 1, 1, 64, 32, dtype="fp32")
    with pytest.raises(blocks.GpannError):
        blocks.Layout(-1, 1, 64, 1, 1, 64, 32)
    with pytest.raises(blocks.GpannError):
        blocks.Layout(1, 1, 1 << 33, 1, 1, 64, 32)


@pytest.mark.parametrize("names,arg,value", [
    ("route attend backward weigh", "q", 0), ("summarize attend backward weigh evict", "k", 0), ("attend backward evict", "v", 0),
    ("route attend backward weigh", "probes", 0), ("summarize route", "summary", 0), ("attend backward", "out", 0), ("backward weigh", "lse", 0),
    ("backward", "dout", 0), ("backward", "dq", 0), ("backward", "dk", 0), ("backward", "dv", 0), ("weigh evict", "mass", 0), ("weigh", "mass_out", 0),
    ("evict", "rows", 0), ("evict", "count", 0), ("evict", "k_out", 0), ("evict", "v_out", 0),
    ("route attend backward weigh", "q", 24), ("summarize attend backward weigh evict", "k", 24), ("attend backward evict", "v", 24), ("route", "summary", 20),
    ("attend backward", "out", 24), ("backward", "dq", 24), ("route attend backward weigh", "probes", 18), ("attend backward weigh", "lse", 18),
    ("weigh evict", "mass", 18), ("evict", "rows", 18), ("evict", "k_out", 40),
    ("route attend backward weigh", "nprobe", 0), ("route attend backward weigh", "nprobe", 65), ("route", "last", 0), ("route", "first", 3), ("route", "last", 5),
    ("route", "last", 0xFFFFFFFF), ("evict", "keep", 0), ("evict", "keep", 2), ("evict", "last", 16), ("evict", "last", 0xFFFFFFFF), ("evict", "k_out", OK),
    ("evict", "mass_out", OK), ("evict", "out_kv_stride", (0, 128, 64)), ("evict", "out_kv_stride", (2048, 64, 64)), ("evict", "out_kv_stride", (2048, 128, 60)),
    ("backward weigh", "workspace", 0), ("backward weigh", "workspace", 24), ("backward weigh", "workspace_bytes", 64)])
def test_arguments_that_are_refused(blocks, names, arg, value):
    L = _layout(blocks)
    for name in names.split():
        _refused(blocks, _calls(blocks, L, **{arg: value})[name])


def test_overlapping_outputs_and_paged_gradients_are_refused(blocks):
    calls = _calls(blocks, _layout(blocks, out_stride=(768, 256, 0)))
    _refused(blocks, calls["attend"], match="overlaps")
    for which in ("q_stride", "k_stride", "v_stride"):
        rows = 256 if which == "q_stride" else 128
        _refused(blocks, _calls(blocks, _layout(blocks, **{which: (0, rows, 64)}))["backward"], match="overlaps")
    _refused(blocks, _calls(blocks, _layout(blocks, page_table=OK, n_pages=4))["backward"], status=5)


def test_a_correct_call_without_a_device_is_an_error(blocks):
    import pygpann
    if pygpann.device_count() > 0:
        pytest.skip("a GPU is present")
    for name, call in _calls(blocks, _layout(blocks)).items():
        _refused(blocks, call, status=2)


def test_workspace_sizes(blocks):
    L = _layout(blocks)
    assert blocks.workspace_bytes(L, 4, []) == 0
    each = {c: blocks.workspace_bytes(L, 4, [c]) for c in blocks.CALLS}
    assert blocks.workspace_bytes(L, 4, list(blocks.CALLS)) == max(each.values())
    _refused(blocks, lambda: blocks.workspace_bytes(L, 65, ["attend"]))
    _refused(blocks, lambda: blocks.workspace_bytes(L, 4, ["scan"]))


def test_reference_gradients_against_differences():
    rng = np.random.default_rng(3)
    g, d, bs, n, scale = 2, 8, 4, 13, 0.3
    q, k, v, dout = rng.normal(size=(g, d)), rng.normal(size=(n, d)), rng.normal(size=(n, d)), rng.normal(size=(g, d))
    probes, vis = [2, 0, 2, -1, 9], 10
    rows, dq, dk, dv, *_ = ref.backward(q, k, v, dout, probes, bs, 4, vis, scale, "bf16")
    assert list(rows) == [0, 1, 2, 3, 8, 9]
    def loss():
        return (ref.attend(q, k, v, probes, bs, 4, vis, scale, "bf16")[0] * dout).sum()
    full_k, full_v = np.zeros_like(k), np.zeros_like(v)
    full_k[rows], full_v[rows] = dk, dv
    for x, grad in ((q, dq), (k, full_k), (v, full_v)):
        for i in np.ndindex(x.shape):
            keep, h = x[i], 1e-5
            x[i] = keep + h
            up = loss()
            x[i] = keep - h
            down = loss()
            x[i] = keep
            assert abs((up - down) / (2 * h) - grad[i]) < 1e-8      # h^2 times third derivatives of order 1, and 1e-16 / h of rounding


@pytest.mark.parametrize("field", ["q_len", "kv_len", "page_table"])
def test_lengths_and_page_tables_have_to_be_aligned(blocks, field):
    L = _layout(blocks, **{field: 18}, n_pages=8)
    for name, call in _calls(blocks, L).items():
        _refused(blocks, call, match="4-byte aligned")


def test_strides_that_would_wrap_are_refused(blocks):
    for bad in (1 << 64, (1 << 63), -(1 << 64)):
        with pytest.raises(blocks.GpannError):
            _layout(blocks, k_stride=(bad, 128, 64))


def test_more_pairs_or_query_rows_than_a_grid_has_room_for_are_refused(blocks):
    many = dict(batch=60000, q_rows=2, kv_rows=16, q_heads=2, kv_heads=2, block_rows=16)
    calls = _calls(blocks, _layout(blocks, **many), workspace_bytes=1 << 40)
    for name in ("backward", "weigh", "route"):
        _refused(blocks, calls[name], match="65535")
    long = dict(batch=1, q_rows=65535 * 128 + 1, kv_rows=16, q_heads=1, kv_heads=1, block_rows=16)
    calls = _calls(blocks, _layout(blocks, **long), workspace_bytes=1 << 40)
    for name in ("backward", "weigh"):
        _refused(blocks, calls[name], match="query rows")
    long = dict(batch=1, q_rows=1 << 22, kv_rows=16 * 4097, q_heads=1, kv_heads=1, block_rows=16)
    _refused(blocks, _calls(blocks, _layout(blocks, **long))["route"], match="query rows")


def test_attention_of_few_tokens_over_long_caches_needs_its_workspace(blocks):
    L = _layout(blocks, batch=1, q_rows=1, kv_rows=4096, block_rows=64)
    need = blocks.workspace_bytes(L, 16, ["attend"])
    assert need > 0 and blocks.workspace_bytes(_layout(blocks, batch=1, q_rows=2000, kv_rows=4096, block_rows=64), 16, ["attend"]) == 0
    for ws in (dict(), dict(workspace=OK, workspace_bytes=need - 1), dict(workspace=24, workspace_bytes=need)):
        _refused(blocks, lambda: blocks.attend(L, OK, OK, OK, OK, 16, OK, **ws), match="workspace")
