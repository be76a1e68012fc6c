"""ngp_gradient_norm / ngp_clip_gradients against 64 bits: many tensors of all three types, odd sizes and addresses, in place and beside, refusals.

Tolerances: the norm is a 64-bit sum rounded to float (2^-24 and a few 2^-52 per thousand additions: 2^-23 covers both); a clipped value is g * c with c a float (2^-24), one 32-bit product (2^-24)
and the rounding to its type (2^-11, 2^-8, 2^-24)."""
import ctypes as C
import math

import numpy as np
import pytest

import ngp_abi as A

U = {A.TYPE_HALF: 2.0 ** -11, A.TYPE_BFLOAT16: 2.0 ** -8, A.TYPE_FLOAT: 2.0 ** -24}
TINY = {A.TYPE_HALF: 2.0 ** -25, A.TYPE_BFLOAT16: 2.0 ** -134, A.TYPE_FLOAT: 2.0 ** -126}  # half a step among the smallest (float: its denormals may count as zero)
H, B, F = A.TYPE_HALF, A.TYPE_BFLOAT16, A.TYPE_FLOAT


def dtype(t):
    import torch
    return {H: torch.float16, B: torch.bfloat16, F: torch.float32}[t]


class Set:
    """tensors inside one marked buffer each, `shift` elements behind its start"""

    def __init__(self, spec, in_place, scale=1.0, shift=1, seed=0):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.items = []
        for n, t in spec:
            buf = torch.full((n + shift + 9,), 33.0, dtype=dtype(t), device="cuda")
            buf[shift:shift + n] = (torch.randn(n, generator=g) * scale).to(dtype(t)).cuda()
            out = buf if in_place else torch.full((n + shift + 9,), 44.0, dtype=dtype(t), device="cuda")
            self.items.append((buf, out, buf[shift:shift + n].clone(), n, t, shift))
        self.in_place = in_place
        size = lambda t: 4 if t == F else 2
        self.table = (A.Gradient * max(1, len(spec)))(*[A.Gradient(b.data_ptr() + s * size(t), o.data_ptr() + s * size(t), n, t, 0) for b, o, _, n, t, s in self.items])
        self.norm = torch.full((3,), -5.0, device="cuda")
        self.ws = torch.full((A.load_hip().ngp_gradient_workspace_size() + 16,), 255, dtype=torch.uint8, device="cuda")

    def exact(self, loss_scale):
        return math.sqrt(math.fsum(float(v.double().square().sum()) for _, _, v, *_ in self.items)) / loss_scale

    def clip(self, loss_scale, max_norm, stream=None):
        L = A.load_hip()
        A.check(L, L.ngp_clip_gradients(stream, len(self.items), self.table, loss_scale, max_norm, self.norm.data_ptr() + 4, self.ws.data_ptr(), self.ws.numel() - 16))

    def check(self, loss_scale, max_norm):
        import torch
        norm = self.exact(loss_scale)
        assert abs(float(self.norm[1]) - norm) <= 2.0 ** -23 * norm and float(self.norm[0]) == -5.0 and float(self.norm[2]) == -5.0
        assert bool((self.ws[-16:] == 255).all())
        c = max_norm / norm if norm > max_norm else 1.0
        for buf, out, v, n, t, s in self.items:
            got, want = out[s:s + n].double(), v.double() * c
            tol = (0 if c == 1.0 else U[t] + 2.0 ** -22) * want.abs() + (0 if c == 1.0 else TINY[t])
            assert bool(((got - want).abs() <= tol).all())
            mark = 33.0 if self.in_place else 44.0
            assert bool((out[:s] == mark).all()) and bool((out[s + n:] == mark).all())
            if not self.in_place:
                assert bool((buf[s:s + n] == v).all())


SPECS = [[(1, H)], [(5, F), (0, H), (7, B)], [(8192, H)], [(8193, B), (8191, F)], [(100003, H), (1, F), (30000, B), (16, H)], [(2_000_001, H)], [(3, H)] * 250 + [(1000, F)] * 40, [(0, F)], []]


@pytest.mark.gpu
@pytest.mark.parametrize("spec", range(len(SPECS)))
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("over", [False, True])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_clip(hip, spec, in_place, over, shift):
    s = Set(SPECS[spec], in_place, shift=shift, seed=spec)
    max_norm = float(np.float32(s.exact(128.0) * (0.3 if over else 1.5)))
    s.clip(128.0, max_norm)
    s.check(128.0, max_norm)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [7, 8, 9, 111, 112, 113])
def test_many_small_tensors(hip, n):
    """either side of the number that one block takes, with empty ones between"""
    s = Set([(40 + 3 * i, (H, F, B)[i % 3]) for i in range(n)] + [(0, F)] * 5, True, seed=n)
    max_norm = float(np.float32(s.exact(2.0) * 0.5))
    s.clip(2.0, max_norm)
    s.check(2.0, max_norm)


@pytest.mark.gpu
@pytest.mark.parametrize("spec", [[(65535, H)], [(65536, B)], [(65537, F)], [(0, H)] * 111 + [(70000, B), (0, F), (9, H)], [(100, H)] * 112 + [(60000, F)], [(8192, B)] * 112 + [(0, F)] * 130 + [(8193, H)] * 3, [(0, F)] * 300 + [(5, H)]])
@pytest.mark.parametrize("in_place", [False, True])
def test_tables(hip, spec, in_place):
    """either side of what one block does alone; tensors over several tables, empty ones at their ends, a table of nothing"""
    s = Set(spec, in_place, shift=1, seed=len(spec))
    max_norm = float(np.float32(s.exact(64.0) * 0.7))
    s.clip(64.0, max_norm)
    s.check(64.0, max_norm)


@pytest.mark.gpu
def test_wide_range(hip):
    """squares beyond and below what 32 bits hold"""
    for scale in (1e30, 1e-30):
        s = Set([(5000, B), (3000, F)], True, scale=scale)
        m = float(np.float32(s.exact(1.0) * 0.5))
        s.clip(1.0, m)
        s.check(1.0, m)


@pytest.mark.gpu
@pytest.mark.parametrize("spec", [[(2, F)], [(3, B), (9, H)], [(300_000, F), (5, B)]])
@pytest.mark.parametrize("loss_scale", [1.0, 2.0 ** -20])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_beyond_the_largest_float(hip, spec, loss_scale, in_place):
    """finite gradients whose norm is no 32-bit number: what is reported is infinite, so the gradients are left as they are"""
    import torch
    s = Set(spec, in_place)
    for buf, out, v, n, t, sh in s.items:
        if t != H:
            v.copy_(torch.where(torch.arange(n, device="cuda") % 2 == 0, 3e38, -3e38).to(v.dtype))
            buf[sh:sh + n] = v
    assert 3.4028235e38 < s.exact(loss_scale) < 1e300
    s.clip(loss_scale, 1e30)
    assert float(s.norm[1]) == float("inf")
    for buf, out, v, n, t, sh in s.items:
        assert bool((out[sh:sh + n] == v).all())


@pytest.mark.gpu
@pytest.mark.parametrize("spec", [[(5, F), (40, B)], [(70_000, F), (8195, B)]])
@pytest.mark.parametrize("scale,loss_scale,max_norm", [(1e35, 1.0, 1e-3), (1e35, 1.0, 1e-7), (1e35, 2.0 ** 60, 1e-21), (1e35, 1.0, 1e-20)])
@pytest.mark.parametrize("in_place", [False, True])
def test_factors_below_the_smallest_float(hip, spec, scale, loss_scale, max_norm, in_place):
    """huge gradients and a small bound: the factor is no 32-bit number in full, the clipped gradients are ordinary ones"""
    s = Set(spec, in_place, scale=scale)
    max_norm = float(np.float32(max_norm))
    assert max_norm / s.exact(loss_scale) < 1.17e-38
    s.clip(loss_scale, max_norm)
    s.check(loss_scale, max_norm)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("t", [H, B, F])
def test_not_finite(hip, bad, t):
    """reported; the gradients stay (in place) or are copied as they are"""
    import torch
    for in_place in (False, True):
        s = Set([(9000, H), (20000, t), (10, F)], in_place)
        buf, out, v, n, _, sh = s.items[1]
        buf[sh + 12345] = bad
        v[12345] = bad
        s.clip(128.0, 1e-3)
        assert not math.isfinite(float(s.norm[1]))
        for buf, out, v, n, _, sh in s.items:
            assert bool(torch.equal(out[sh:sh + n].nan_to_num(nan=1.5), v.nan_to_num(nan=1.5)))


@pytest.mark.gpu
def test_counted_but_not_clipped(hip):
    s = Set([(4000, H), (5000, F)], False)
    s.table[1].clipped = None
    m = float(np.float32(s.exact(1.0) * 0.25))
    s.clip(1.0, m)
    assert bool((s.items[1][1] == 44.0).all())
    want = s.items[0][2].double() * 0.25
    assert bool(((s.items[0][1][1:4001].double() - want).abs() <= (U[H] + 2.0 ** -22) * want.abs() + TINY[H]).all())


@pytest.mark.gpu
def test_max_norm_zero_and_infinite(hip):
    s = Set([(4000, H), (5000, F)], True)
    s.clip(1.0, float("inf"))
    s.check(1.0, float("inf"))
    s.clip(1.0, 0.0)
    assert all(bool((o[1:1 + n] == 0).all()) for _, o, _, n, _, _ in s.items)


@pytest.mark.gpu
def test_clipped_norm_is_the_bound(hip):
    s = Set([(100_000, F), (77_777, F)], True)
    L = A.load_hip()
    s.clip(2.0, 3.0)
    A.check(L, L.ngp_gradient_norm(None, 2, s.table, 2.0, s.norm.data_ptr(), s.ws.data_ptr(), s.ws.numel()))
    assert abs(float(s.norm[0]) - 3.0) <= 3.0 * 2.0 ** -21


@pytest.mark.gpu
def test_graph_and_stream(hip):
    """captured once (the table is in the launch), replayed over new gradients with other work between; on a stream of its own"""
    import torch
    s = Set([(50_000, H), (300_001, B), (7000, F)], True)
    L = A.load_hip()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.clip(128.0, 0.5, torch.cuda.current_stream().cuda_stream)
    C.memset(s.table, 0, C.sizeof(s.table))  # the caller's table is free to go
    for k in range(4):
        for buf, _, v, n, t, sh in s.items:
            v.copy_((torch.randn(n, device="cuda") * 10.0 ** k).to(dtype(t)))
            buf[sh:sh + n] = v
        s.ws[:-16].fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        s.check(128.0, 0.5)
    s = Set([(50_000, H)], True)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    s.clip(1.0, 0.5, st.cuda_stream)
    st.synchronize()
    s.check(1.0, 0.5)


@pytest.mark.gpu
def test_same_bits_every_time(hip):
    got = []
    for _ in range(3):
        s = Set([(1_500_000, H), (200_000, F)], False, seed=4)
        s.clip(128.0, 0.1)
        got.append((s.norm.clone(), [o.clone() for _, o, *_ in s.items]))
    for n, o in got[1:]:
        assert bool((n == got[0][0]).all()) and all(bool((a == b).all()) for a, b in zip(o, got[0][1]))


def test_refusals():
    L = A.load_hip()

    def call(tensors, loss_scale=1.0, max_norm=1.0, norm=0x100000, ws=0x200000, size=1 << 20, n=None, f="clip"):
        table = (A.Gradient * max(1, len(tensors)))(*[A.Gradient(*t) for t in tensors])
        n = len(tensors) if n is None else n
        rc = L.ngp_clip_gradients(None, n, table, loss_scale, max_norm, norm, ws, size) if f == "clip" else L.ngp_gradient_norm(None, n, table, loss_scale, norm, ws, size)
        assert rc != 0
        return L.ngp_last_error().decode()
    good = (0x1000, 0x1000, 16, H, 0)
    assert "type" in call([(0x1000, 0x1000, 16, 3, 0)])
    assert "null gradient" in call([(None, 0x1000, 16, H, 0)])
    assert "aligned" in call([(0x1001, 0x1001, 16, H, 0)]) and "aligned" in call([(0x1002, 0x1002, 16, F, 0)]) and "aligned" in call([(0x1000, 0x2001, 16, H, 0)])
    assert "norm" in call([good], norm=0x100002) and "null" in call([good], norm=None)
    assert "workspace" in call([good], ws=None) and "workspace" in call([good], size=100) and "workspace" in call([good], ws=0x200008)
    for v in (0.0, -1.0, float("nan"), float("inf")):
        assert "loss_scale" in call([good], loss_scale=v)
    for v in (-1.0, float("nan")):
        assert "max_norm" in call([good], max_norm=v)
    assert "overlaps" in call([good, good])                                                     # the same tensor twice, in place
    assert "overlaps" in call([(0x1000, 0x3000, 16, H, 0), (0x2000, 0x3010, 16, H, 0)])          # two outputs
    assert "overlaps" in call([(0x1000, 0x1010, 16, H, 0)])                                     # half in place
    assert "overlaps" in call([(0x1000, 0x2000, 16, H, 0), (0x2000, 0x4000, 16, H, 0)])          # an output on another input
    assert "overlaps" in call([(0x200000, 0x200000, 16, H, 0)]) and "overlaps" in call([(0x100000, 0x100000, 16, F, 0)])
    if not L.ngp_device_available():
        ok = [good, (0x1020, 0x1020, 16, H, 0), (0x4000, 0x5000, 3, F, 0), (None, None, 0, B, 0)]
        assert "no HIP device" in call(ok) and "no HIP device" in call(ok[::-1]) and "no HIP device" in call([good, good], f="norm")  # (the norm may count a tensor twice)


def test_norm_does_not_look_at_clipped():
    """ngp_gradient_norm takes a table whose `clipped` was never set: whatever stands there is no reason to refuse it"""
    L = A.load_hip()
    if L.ngp_device_available():
        pytest.skip("has a GPU: these addresses are not its own")
    for clipped in (0x2001, 0x1001, 0x100000, 0x200000, 0x1008, (1 << 64) - 1):
        table = (A.Gradient * 2)(A.Gradient(0x1000, clipped, 16, H, 0), A.Gradient(0x4000, clipped, 16, F, 0))
        assert L.ngp_gradient_norm(None, 2, table, 1.0, 0x100000, 0x200000, 1 << 20) != 0
        assert "no HIP device" in L.ngp_last_error().decode()
