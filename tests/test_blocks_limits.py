"""CPU: refusals of the block operators at the ends of their ranges — before anything is enqueued, and before a number would wrap."""
import pytest

from test_blocks_refusals import OK, _calls, _layout, _refused, blocks   # noqa: F401  (blocks: the fixture)


def test_gradients_of_more_workgroups_than_a_launch_has_room_for_are_refused_before_the_first(blocks):
    """600 pairs of 16384 blocks: the query side would fit, the key side has 9.8 million workgroups"""
    L = _layout(blocks, batch=600, q_rows=2, kv_rows=16384 * 16, q_heads=1, kv_heads=1, block_rows=16)
    _refused(blocks, _calls(blocks, L, workspace_bytes=1 << 45)["backward"], status=5, match="workgroups")


@pytest.mark.parametrize("strides", [(256, 64), (256, 64, 64, 64), (64,)])
@pytest.mark.parametrize("which", ["q_stride", "k_stride", "v_stride", "out_stride"])
def test_strides_are_three_numbers(blocks, which, strides):
    with pytest.raises(blocks.GpannError, match="three"):
        _layout(blocks, **{which: strides})


@pytest.mark.parametrize("value", [-1, 1 << 64, (1 << 64) + 4096])
def test_workspace_sizes_that_would_wrap_are_refused(blocks, value):
    L = _layout(blocks)
    for name in ("backward", "weigh"):
        _refused(blocks, _calls(blocks, L, workspace_bytes=value)[name], match="workspace_bytes")
    ws = dict(workspace=OK, workspace_bytes=value)
    for call in (lambda: blocks.route(L, OK, OK, 4, OK, **ws), lambda: blocks.attend(L, OK, OK, OK, OK, 4, OK, **ws),
                 lambda: blocks.evict(L, OK, OK, OK, 16, OK, OK, 32, 48, 64, **ws)):
        _refused(blocks, call, match="workspace_bytes")


@pytest.mark.parametrize("strides", [((1 << 64) + 2048, 128, 64), (2048, 128), (2048, 128, 64, 8), (-(1 << 64) + 2048, 128, 64)])
def test_strides_of_evicted_caches_that_would_wrap_are_refused(blocks, strides):
    _refused(blocks, _calls(blocks, _layout(blocks), out_kv_stride=strides)["evict"], match="three")


@pytest.mark.parametrize("device", [1 << 32, -(1 << 32), 1 << 31])
def test_devices_that_would_wrap_are_refused(blocks, device):
    with pytest.raises(blocks.GpannError, match="device"):
        _layout(blocks, device=device)


@pytest.mark.parametrize("pointer", [1 << 64, -16])
def test_pointers_that_would_wrap_are_refused(blocks, pointer):
    _refused(blocks, lambda: blocks.attend(_layout(blocks), pointer, OK, OK, OK, 4, OK), match="pointer")
    with pytest.raises(blocks.GpannError, match="pointer"):
        _layout(blocks, kv_len=pointer)


@pytest.mark.parametrize("scale", [3e38, -2.5e38])
def test_scales_whose_powers_of_two_are_not_finite_are_refused(blocks, scale):
    """the kernels' exponentials are powers of two: of the logits times log2 e = 1.44"""
    for name, call in _calls(blocks, _layout(blocks, scale=scale)).items():
        _refused(blocks, call, match="scale")
