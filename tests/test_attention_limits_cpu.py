"""How large an attention call may be: more workgroups than a launch counts are refused
on the host, before any device call."""
import pytest

from spar_amd import hip

A = 1 << 20  # an address that is never read
NO_DEVICE = 999  # calls that pass the checks end here


def heads():
    return hip.heads(A, (64, 64, 64))


def shape(batch, queries, keys, sinks=0, window=0):
    return hip.attention(batch, 8, 8, queries, keys, 8, window, sinks, 1.0, None, hip.INT32, 0)


def forward(call):
    need = hip.attention_workspace(call, 0)
    return hip.status_of("spar_hip_launch_attention_forward", heads(), None, heads(), heads(),
                         heads(), call, A, need, NO_DEVICE).code


def backward(call):
    need = hip.attention_workspace(call, 1)
    return hip.status_of("spar_hip_launch_attention_backward", *[heads()] * 5, A, *[heads()] * 3,
                         call, A, need, NO_DEVICE).code


@pytest.mark.parametrize("batch,queries,keys", [(1 << 21, 1, 1), (1 << 20, 65, 1),
                                                (1 << 18, 500, 500), (1 << 27, 1, 1)])
def test_more_workgroups_than_a_launch_counts_are_refused(batch, queries, keys):
    call = shape(batch, queries, keys)
    assert forward(call) == 1
    assert backward(call) == 1


def test_sixteen_rows_a_workgroup():
    call = shape(1 << 20, 17, 1)  # two workgroups of the forward, one of the backward
    assert forward(call) == 1
    assert backward(call) not in (0, 1)


def test_tiles_of_keys_count_too():
    assert backward(shape(1 << 18, 1, 500)) == 1
    assert backward(shape(1 << 19, 1, 190, sinks=64, window=1)) == 1


def test_fewer_pass_the_checks():
    call = shape((1 << 21) - 1, 1, 1)
    assert forward(call) not in (0, 1) and backward(call) not in (0, 1)
