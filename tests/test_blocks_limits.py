"""CPU: refusals of the block operators at the ends of their ranges — before anything is enqueued."""
from test_blocks_refusals import _calls, _layout, _refused, blocks   # noqa: F401  (blocks: the fixture)


def test_gradients_of_more_workgroups_than_a_launch_has_room_for_are_refused_before_the_first(blocks):
    """600 pairs of 16384 blocks: the query side would fit, the key side has 9.8 million workgroups"""
    L = _layout(blocks, batch=600, q_rows=2, kv_rows=16384 * 16, q_heads=1, kv_heads=1, block_rows=16)
    _refused(blocks, _calls(blocks, L, workspace_bytes=1 << 45)["backward"], status=5, match="workgroups")
