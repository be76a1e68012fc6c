"""Dense layers near the limits of a launch: every call is refused before anything is launched, or asks for grids that the runtime takes."""
import pytest

import ngp_abi as A
import played_runtime

CALLS = """
import itertools
runtime.devices(1)
at = lambda i: (i + 1) << 42


def call(gated, backward, m, n, k, want="xwb", act=A.ACT_RELU):
    # (linear activations, so that nothing depends on what the buffers hold); True: accepted
    size = (L.ngp_gated_workspace_size if gated else L.ngp_linear_workspace_size)(m, n, k, backward)
    ws = (at(20) if size else None, size)
    x, w, dx, dw, db = at(0), at(1), at(6) if "x" in want else None, at(7) if "w" in want else None, at(9) if "b" in want else None
    if gated and backward:
        args = (k, w, at(2), k, at(4), at(5), n, at(8), n, dx, k, dw, dw and at(10), k, db, db and at(11))
    elif gated:
        args = (k, w, at(2), k, None, None, at(3), n, at(4), at(5), n)
    elif backward:
        args = (k, w, k, at(4), n, at(8), n, dx, k, dw, k, db)
    else:
        args = (k, w, k, None, None, 0, at(3), n, at(4), n)
    before, bad = runtime.launches(), runtime.launches_out_of_range()
    f = {(0, 0): L.ngp_linear_forward, (0, 1): L.ngp_linear_backward, (1, 0): L.ngp_gated_forward, (1, 1): L.ngp_gated_backward}[gated, backward]
    rc = f(None, A.TYPE_HALF, act, m, n, k, x, *args, *ws)
    assert runtime.launches_out_of_range() == bad, (gated, backward, m, n, k, want)
    if rc:
        assert runtime.launches() == before and "tiles" in L.ngp_last_error().decode(), (gated, backward, m, n, k, want, L.ngp_last_error())
    return rc == 0


big = (1 << 31) - 1
"""

TILES = CALLS + """
for gated in (0, 1):
    for m, n, k in ((big, 1, 1), (big, 7, 1), (big, 1, 7), (big - 127, 1, 1), (big - 255, 1, 1), (big // 2 + 1, 65, 1), (1 << 30, 130, 4), (big, 64, 1), (big, 8, 8), (big, 16, 16), (40, 1 << 24, 300), (1 << 20, 1 << 17, 9)):
        for backward, want in ((0, ""), (1, "xwb"), (1, "x"), (1, "w"), (1, "b"), (1, "")):
            call(gated, backward, m, n, k, want)
    # what fits stays accepted: a launch of 2^24 - 1 tiles, narrow layers, gradients of the weights and biases alone
    assert call(gated, 0, big - 255, 1, 1) and call(gated, 0, big, 8, 8) and call(gated, 1, big, 8, 8)
    assert call(gated, 1, big, 1, 1, "w") and call(gated, 1, big, 1, 1, "b") and call(gated, 1, big, 1, 1, "wb")
    assert not call(gated, 0, big, 1, 1) and not call(gated, 1, big, 1, 1, "x") and not call(gated, 1, big, 1, 1)
print("done")
"""

COPIES = CALLS + """
# lines that are no whole pieces, 64 GB of them: copied before the products, more 16-byte pieces than a launch has threads
for gated, m, n, k in ((0, 16500, 768, (1 << 21) - 1), (1, 20000, 500, (1 << 21) - 1), (0, 40000000, 800, 1003), (0, 16500, 900, (1 << 21) - 3)):
    for backward in (0, 1):
        assert call(gated, backward, m, n, k)
print("done")
"""


@pytest.mark.parametrize("calls", [TILES, COPIES], ids=["tiles", "copies"])
def test_grids(calls, tmp_path):
    if A.load_hip().ngp_device_available():
        pytest.skip("has a GPU: the runtime is not to be played there")
    played_runtime.run(calls, tmp_path)
