"""Attention calls whose sizes pass what 32 bits or one launch can count."""
import numpy as np
import pytest

from tests.attention_oracle import assert_within, half_step
from tests.test_attention_gpu import F32, F64, _alive, _release_buffers, device, space  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keys,extent,batch", [
    ((1 << 24) + 100, 256, 1),  # a key head of more than 2^32 elements
    (8200, 256, 260),           # and many that one launch cannot join
])
def test_gradients_of_many_sinks(hip, keys, extent, batch):
    """Two queries that see every key as a sink, all keys and values one vector: weights
    are 1 / n, and dv of key j is the sum of g / n over the queries that see it.  Keys and
    values have a token stride of 0; their gradients and the workspace take 69 GB where
    there is one sequence."""
    rng = np.random.default_rng(31)
    key, value = rng.standard_normal((2, extent)).astype(F32)
    q, g = rng.standard_normal((2, batch, 2, extent)).astype(F32)
    output = np.broadcast_to(value, (batch, 2, extent))
    shape = hip.attention(batch, 1, 1, 2, keys, extent, 1, keys, 0.1, None, hip.INT32, 0)
    of_rows = (2 * extent, 0, extent)
    rows = [hip.heads(device(hip, x).ptr, of_rows) for x in (g, output, q)]
    one = [hip.heads(device(hip, x).ptr, (0, 0, 0)) for x in (key, value)]
    dq = space(hip, batch * 2 * extent * 4)
    made = [space(hip, batch * keys * extent * 4) for _ in range(2)]
    need = hip.attention_workspace(shape, 1)
    logsumexp = device(hip, (0.1 * (q @ key) + np.log([keys - 1, keys])).astype(F32))
    of_keys = (keys * extent, 0, extent)
    hip.call("spar_hip_launch_attention_backward", hip.heads(dq.ptr, of_rows),
             *(hip.heads(x.ptr, of_keys) for x in made), rows[0], rows[1], logsumexp.ptr, rows[2],
             *one, shape, space(hip, need).ptr, need, 0)
    weight = np.array([1 / (keys - 1), 1 / keys])
    u = half_step(F32)
    # dP and delta are one sum of products formed twice, delta of an output that is exact
    size = 2 * (np.abs(g) @ np.abs(value)).astype(F64)
    for b in sorted({0, batch // 2, batch - 1}):
        for j in sorted({0, 5, 63, 64, keys // 2, keys - 101, keys - 99, keys - 2, keys - 1}):
            seen = np.array([j < keys - 1, True])
            got = []
            for x in made:
                row = np.empty(extent, F32)
                hip.call("spar_hip_copy_device_to_host", row.ctypes.data,
                         x.address((b * keys + j) * extent * 4), row.nbytes, 0)
                got.append(row)
            share = (weight * seen)[:, None]
            # sums of up to 2^14 equal weights in a lane, and those of lanes and parts
            assert_within(got[1], (share * g[b]).sum(0), ((1 << 14) + 64) * u *
                          (share * np.abs(g[b])).sum(0), f"dv of {b}, {j}")
            assert_within(got[0], np.zeros(extent), 0.1 * (extent + 64) * u *
                          (share * size[b][:, None] * np.abs(q[b])).sum(0), f"dk of {b}, {j}")
    _alive.clear()
    hip.call("spar_hip_empty_cache", 0)
