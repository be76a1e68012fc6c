"""Dense layers and gradient clipping with several devices in sight: what lies on another device than the current one is refused before anything is launched."""
import pytest

import ngp_abi as A
import played_runtime

CALLS = """
FAR = 1 << 40
at = lambda i: 0x1000000 + (i << 16)


def refused(f, args, what):
    before = runtime.launches()
    assert f(*args) != 0 and what in L.ngp_last_error().decode(), (what, L.ngp_last_error())
    assert runtime.launches() == before


def calls(f, names, args):
    # accepted as it stands; refused with any one buffer on the other device or at no device's address, and with the other device's stream
    before = runtime.launches()
    assert f(*args) == 0, L.ngp_last_error()
    assert runtime.launches() > before
    for i, name in names.items():
        for address, what in ((FAR + args[i], " lies on another device"), (0x2000, " is not a device pointer")):
            refused(f, list(args[:i]) + [address] + list(args[i + 1:]), name + what)
    refused(f, [3] + list(args[1:]), "stream")
    assert f(2, *args[1:]) == 0


n_ws = 1 << 20
calls(L.ngp_linear_forward, {6: "x", 8: "w", 10: "bias", 11: "residual", 13: "y", 15: "pre", 17: "workspace"},
      [None, 0, 1, 2, 16, 8192, at(0), 8192, at(1), 8192, at(8), at(9), 16, at(10), 16, at(11), 16, at(12), n_ws])
calls(L.ngp_linear_backward, {6: "x", 8: "w", 10: "pre", 12: "dy", 14: "dx", 16: "dw", 18: "dbias", 19: "workspace"},
      [None, 0, 1, 8, 16, 32, at(0), 32, at(1), 32, at(2), 16, at(3), 16, at(4), 32, at(5), 32, at(6), at(7), n_ws])
calls(L.ngp_gated_forward, {6: "x", 8: "w_gate", 9: "w_up", 11: "bias_gate", 12: "bias_up", 13: "y", 15: "gate_pre", 16: "up_pre"},
      [None, 1, 4, 8, 16, 32, at(0), 32, at(1), at(2), 32, at(3), at(4), at(5), 16, at(6), at(7), 16, None, 0])
calls(L.ngp_gated_backward, {6: "x", 8: "w_gate", 9: "w_up", 11: "gate_pre", 12: "up_pre", 14: "dy", 16: "dx", 18: "dw_gate", 19: "dw_up", 21: "dbias_gate", 22: "dbias_up", 23: "workspace"},
      [None, 1, 4, 8, 16, 32, at(0), 32, at(1), at(2), 32, at(3), at(4), 16, at(5), 16, at(6), 32, at(7), at(8), 32, at(9), at(10), at(11), n_ws])


def clip(stream, grad, clipped, norm, workspace, both=True):
    table = (A.Gradient * 2)(A.Gradient(grad, clipped, 100, 0, 0), A.Gradient(at(20), at(20), 100, 2, 0))
    return L.ngp_clip_gradients(stream, 2, table, 1.0, 1.0, norm, workspace, n_ws) if both else L.ngp_gradient_norm(stream, 2, table, 1.0, norm, workspace, n_ws)


ws = 1 << 30
calls(clip, {1: "a gradient", 2: "a clipped gradient", 3: "norm", 4: "workspace"}, [None, at(0), at(1), at(2), ws])
calls(lambda *a: clip(*a, both=False), {1: "a gradient", 3: "norm", 4: "workspace"}, [None, at(0), at(1), at(2), ws])
print("done")
"""


def test_other_devices_are_refused(tmp_path):
    if A.load_hip().ngp_device_available():
        pytest.skip("has a GPU: the runtime is not to be played there")
    played_runtime.run(CALLS, tmp_path)
