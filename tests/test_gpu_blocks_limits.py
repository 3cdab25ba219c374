"""GPU: where the block operators' ranges end — values that are not numbers in rows a key is hidden from, weights and gradients at the ends of
binary16, log-sum-exps of more keys than a call's, strides and sizes beyond the usual ones — against their definitions in binary64."""
import pytest
import torch

from test_gpu_blocks import Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def blocks(gp):
    from pygpann import blocks
    return blocks


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
