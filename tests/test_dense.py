"""Dense layers (ngp_linear_*, ngp_gated_*): forward and backward against a plain computation in 64 bits, refusals, streams, graphs, and a network of them trained end to end.

Tolerances.  With u = eps / 2 of the type (half 2^-11, bfloat16 2^-8) an output of the forward pass is the exact value rounded once (u |v|), moved by what 32-bit sums lose:
every product sum carries at most (k + 8) 2^-24 sum|x w| (k additions in some order, a bias, the activation's own few operations), and an activation passes a change of its argument
on with a slope of at most 1.2 (none, relu, logistic, silu, gelu) or its own value (exponential).  The backward pass rounds G once between the products: u sum|g w| on top of the sum's bound.
Activations in 32 bits (v_exp_f32, v_rcp_f32, erfcf: a few units in the last place) are covered by 64 * 2^-24 relative to 1 + |value|."""
import ctypes as C
import math

import numpy as np
import pytest

import ngp_abi as A

U = {A.TYPE_HALF: 2.0 ** -11, A.TYPE_BFLOAT16: 2.0 ** -8}
TINY = {A.TYPE_HALF: 2.0 ** -25, A.TYPE_BFLOAT16: 2.0 ** -134}  # half a step among the type's smallest numbers
ACTS = [A.ACT_NONE, A.ACT_RELU, A.ACT_LOGISTIC, A.ACT_EXPONENTIAL, A.ACT_SILU, A.ACT_GELU]
F32 = 2.0 ** -24


def lib():
    return A.load_hip()


def act64(act, z):
    """(act(z), act'(z)) in 64 bits"""
    import torch
    one = torch.ones_like(z)
    if act == A.ACT_NONE:
        return z, one
    if act == A.ACT_RELU:
        return torch.where(z < 0, 0 * one, z), torch.where(z > 0, one, 0 * one)
    if act == A.ACT_EXPONENTIAL:
        return z.exp(), z.exp()
    if act == A.ACT_GELU:
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    p, q = torch.sigmoid(z), torch.sigmoid(-z)
    return (p, p * q) if act == A.ACT_LOGISTIC else (z * p, p + z * p * q)


class Layer:
    """One layer's buffers on the GPU, inside larger ones filled with NaN (nothing beside a matrix may be read into a result) and, for outputs, with a mark (nothing beside them is written)."""
    MARK = 77.0

    def __init__(self, type_, act, m, n, k, gated=False, bias=True, residual=False, pad=(0, 0, 0), shift=0, seed=0, x_scale=1.0):
        import torch
        self.t, self.type, self.act, self.m, self.n, self.k, self.gated = torch, type_, act, m, n, k, gated
        self.dtype = torch.float16 if type_ == A.TYPE_HALF else torch.bfloat16
        self.shift, self.outs = shift, []
        g = torch.Generator().manual_seed(1000 * seed + 7 * m + 3 * n + k)
        s = math.sqrt(2.0 / max(1, n + k))
        self.x = self.matrix(torch.randn(m, k, generator=g) * x_scale, pad[0])
        self.w = [self.matrix(torch.randn(n, k, generator=g) * s, pad[1]) for _ in range(2 if gated else 1)]
        self.bias = [self.matrix(torch.randn(1, n, generator=g) * 0.3, 0) if bias else None for _ in self.w]
        self.residual = self.matrix(torch.randn(m, n, generator=g), pad[2]) if residual else None
        self.dy = self.matrix(torch.randn(m, n, generator=g) * 2.0 ** -4, pad[2])
        self.pad = pad

    def place(self, rows, cols, pad, fill):
        """rows x cols inside a buffer: `shift` elements in front (16 bytes kept), `pad` behind each row, some behind the last"""
        b = self.t.full((8 + self.shift + rows * (cols + pad) + 64,), fill, dtype=self.dtype, device="cuda")
        return b, b[8 + self.shift:8 + self.shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] if rows * (cols + pad) else b[:0].view(rows, cols)

    def matrix(self, values, pad):
        b, v = self.place(values.shape[0], values.shape[1], pad, float("nan"))
        v.copy_(values.to(self.dtype).cuda())
        return b, v

    def out(self, rows, cols, pad=0):
        b, v = self.place(rows, cols, pad, self.MARK)
        self.outs.append((b, v, rows, cols, pad))
        return b, v

    def p(self, bv):
        return None if bv is None else bv[0].data_ptr() + 2 * (8 + self.shift)

    def untouched(self):
        for b, v, rows, cols, pad in self.outs:
            c = b.clone()
            if rows * (cols + pad):
                c[8 + self.shift:8 + self.shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] = self.MARK
            assert bool((c == self.MARK).all()), "written beside an output"

    def z64(self):
        return [self.x[1].double() @ w[1].double().t() + (b[1].double() if b else 0) for w, b in zip(self.w, self.bias)]

    def z_abs(self):
        return [self.x[1].double().abs() @ w[1].double().abs().t() + (b[1].double().abs() if b else 0) for w, b in zip(self.w, self.bias)]

    def forward(self, save=True, stream=None, y_is_residual=False):
        L, m, n, k = lib(), self.m, self.n, self.k
        y = self.residual if y_is_residual else self.out(m, n, self.pad[2])
        pre = [self.out(m, n, self.pad[2]) if save else None for _ in self.w]
        ws = self.workspace(0)
        xs, wst, ns = k + self.pad[0], k + self.pad[1], n + self.pad[2]
        if self.gated:
            rc = L.ngp_gated_forward(stream, self.type, self.act, m, n, k, self.p(self.x), xs, self.p(self.w[0]), self.p(self.w[1]), wst, self.p(self.bias[0]), self.p(self.bias[1]),
                                     self.p(y), ns, self.p(pre[0]), self.p(pre[1]), ns, *ws)
        else:
            rc = L.ngp_linear_forward(stream, self.type, self.act, m, n, k, self.p(self.x), xs, self.p(self.w[0]), wst, self.p(self.bias[0]), self.p(self.residual), ns,
                                      self.p(y), ns, self.p(pre[0]), ns, *ws)
        A.check(L, rc)
        return y, pre

    def workspace(self, backward):
        size = (lib().ngp_gated_workspace_size if self.gated else lib().ngp_linear_workspace_size)(self.m, self.n, self.k, backward)
        self.ws = self.t.full((size + 64,), 255, dtype=self.t.uint8, device="cuda")  # (all ones: NaN in every type)
        return self.ws.data_ptr(), size

    def backward(self, pre, want="xwb", stream=None):
        L, m, n, k = lib(), self.m, self.n, self.k
        dx = self.out(m, k, self.pad[0]) if "x" in want else None
        dw = [self.out(n, k, self.pad[1]) if "w" in want else None for _ in self.w]
        db = [self.out(1, n) if "b" in want else None for _ in self.w]
        xs, wst, ns = k + self.pad[0], k + self.pad[1], n + self.pad[2]
        ws = self.workspace(1)
        if self.gated:
            rc = L.ngp_gated_backward(stream, self.type, self.act, m, n, k, self.p(self.x), xs, self.p(self.w[0]), self.p(self.w[1]), wst, self.p(pre[0]), self.p(pre[1]), ns, self.p(self.dy), ns,
                                      self.p(dx), xs, self.p(dw[0]), self.p(dw[1]), wst, self.p(db[0]), self.p(db[1]), *ws)
        else:
            rc = L.ngp_linear_backward(stream, self.type, self.act, m, n, k, self.p(self.x), xs, self.p(self.w[0]), wst, self.p(pre[0]), ns, self.p(self.dy), ns,
                                       self.p(dx), xs, self.p(dw[0]), wst, self.p(db[0]), *ws)
        A.check(L, rc)
        assert bool((self.ws[ws[1]:] == 255).all()), "written behind the workspace"
        return dx, dw, db

    def close(self, got, want, bound, what):
        u = U[self.type]
        tol = u * want.abs() + (1 + u) * bound + TINY[self.type]
        bad = ~((got.double() - want).abs() <= tol)
        assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() / tol).max()):.2f} of the tolerance"

    def check_forward(self, y, pre):
        z, za = self.z64(), self.z_abs()
        dz = [(self.k + 8) * F32 * v for v in za]
        for p, v, d in zip(pre, z, dz):
            if p is not None:
                self.close(p[1], v, d, "pre")
        a = act64(self.act, z[0])[0]
        da = dz[0] * (1.2 if self.act != A.ACT_EXPONENTIAL else a * 1.01 + 0 * a) + 64 * F32 * (1 + a.abs())
        if self.gated:
            want = a * z[1]
            bound = da * z[1].abs() + a.abs() * dz[1] + da * dz[1] + 2 * F32 * want.abs()
        else:
            want = a + (self.residual64 if self.residual is not None else 0)
            bound = da + 2 * F32 * (a.abs() + want.abs())
        self.close(y[1], want, bound, "y")

    def check_backward(self, pre, dx, dw, db, g_rounding=None):
        z = [p[1].double() for p in pre]
        value, slope = act64(self.act, z[0])
        dy = self.dy[1].double()
        g = [dy * slope * z[1], dy * value] if self.gated else [dy * slope]
        # G: a few 32-bit operations (slopes of magnitude <= 1.2 or the value itself), then one rounding
        fine = [64 * F32 * (v.abs() + (dy * (z[1] if self.gated else 1)).abs()) if i == 0 else 64 * F32 * (v.abs() + dy.abs()) for i, v in enumerate(g)]
        off = [(U[self.type] if g_rounding is None else g_rounding) * v.abs() + f + TINY[self.type] for v, f in zip(g, fine)]
        x, w = self.x[1].double(), [v[1].double() for v in self.w]
        if dx is not None:
            want = sum(a @ b for a, b in zip(g, w))
            size = sum((a.abs() + o) @ b.abs() for a, o, b in zip(g, off, w))
            self.close(dx[1], want, sum(o @ b.abs() for o, b in zip(off, w)) + (2 * self.n + 8) * F32 * size, "dx")
        for a, o, f, d, b in zip(g, off, fine, dw, db):
            if d is not None:
                self.close(d[1], a.t() @ x, o.t() @ x.abs() + (self.m + 8) * F32 * ((a.abs() + o).t() @ x.abs()), "dw")
            if b is not None:
                self.close(b[1][0], a.sum(0), f.sum(0) + (self.m + 8) * F32 * a.abs().sum(0), "dbias")


def run_layer(layer, save=True, backward=True, want="xwb"):
    layer.residual64 = layer.residual[1].double().clone() if layer.residual is not None else None
    y, pre = layer.forward(save)
    layer.check_forward(y, pre)
    if backward:
        layer.check_backward(pre, *layer.backward(pre, want))
    layer.untouched()


SIZES = [(1, 1, 1), (1, 64, 64), (2, 3, 5), (7, 16, 31), (16, 16, 16), (17, 130, 63), (33, 8, 200), (64, 64, 64), (100, 129, 127), (129, 257, 65), (128, 128, 128), (300, 72, 520), (1, 1000, 1000), (5, 264, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [A.TYPE_HALF, A.TYPE_BFLOAT16])
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("gated", [False, True])
def test_sizes(hip, type_, m, n, k, gated):
    run_layer(Layer(type_, A.ACT_SILU if gated else A.ACT_GELU, m, n, k, gated=gated, residual=not gated))


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [A.TYPE_HALF, A.TYPE_BFLOAT16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_activations(hip, type_, act, gated, bias):
    run_layer(Layer(type_, act, 150, 136, 96, gated=gated, bias=bias, residual=not bias and not gated), want="xwb" if bias else "xw")


@pytest.mark.gpu
@pytest.mark.parametrize("pad,shift", [((8, 8, 8), 0), ((1, 3, 5), 0), ((0, 0, 0), 1), ((8, 0, 3), 3), ((5, 8, 0), 4), ((0, 1, 0), 0), ((3, 0, 0), 0)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(70, 90, 64), (257, 136, 200), (9, 40, 129), (1, 96, 72)])
def test_strides_and_alignment(hip, pad, shift, gated, m, n, k):
    run_layer(Layer(A.TYPE_HALF, A.ACT_SILU, m, n, k, gated=gated, residual=not gated, pad=pad, shift=shift))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(0, 5, 7), (5, 0, 7), (5, 7, 0), (0, 0, 0)])
@pytest.mark.parametrize("gated", [False, True])
def test_empty(hip, m, n, k, gated):
    """no samples: gradients of the weights are zero; no inputs: the layer is act(bias) + residual; no outputs: dx is zero"""
    run_layer(Layer(A.TYPE_HALF, A.ACT_SILU, m, n, k, gated=gated, residual=not gated))


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [A.TYPE_HALF, A.TYPE_BFLOAT16])
@pytest.mark.parametrize("m,n,k,gated", [(5000, 64, 64, False), (40001, 40, 24, False), (9000, 256, 256, False), (4099, 200, 136, True), (1500, 777, 500, False), (2048, 512, 1024, True),
                                         (513, 1032, 264, False), (20000, 256, 63, False)])
def test_larger(hip, type_, m, n, k, gated):
    """sums split over blocks, several tiles each way"""
    run_layer(Layer(type_, A.ACT_RELU if not gated else A.ACT_GELU, m, n, k, gated=gated))


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_parts_of_the_gradient(hip, gated):
    """each output alone is bit for bit the one of the whole call"""
    layer = Layer(A.TYPE_HALF, A.ACT_SILU, 700, 136, 72, gated=gated)
    _, pre = layer.forward()
    whole = layer.backward(pre)
    for want, pick in (("x", lambda r: [r[0]]), ("w", lambda r: r[1]), ("b", lambda r: r[2])):
        part = layer.backward(pre, want)
        for a, b in zip(pick(part), pick(whole)):
            assert bool((a[1] == b[1]).all())
    layer.backward(pre, "")
    layer.untouched()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 200])
def test_residual_in_place(hip, m):
    layer = Layer(A.TYPE_HALF, A.ACT_GELU, m, 130, 64, residual=True, pad=(0, 0, 6))
    layer.residual64 = layer.residual[1].double().clone()
    y, pre = layer.forward(y_is_residual=True)
    layer.check_forward(y, pre)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_columns_of_one_buffer(hip, m):
    """input and output as columns of one wider matrix (a concatenation without a copy)"""
    import torch
    L, n, k = lib(), 72, 64
    buf = torch.randn(m, k + n + 8, device="cuda").half()
    w = (torch.randn(n, k, device="cuda") / 8).half()
    want = (buf[:, :k].double() @ w.double().t()).relu()
    tail = buf[:, k + n:].clone()
    A.check(L, L.ngp_linear_forward(None, A.TYPE_HALF, A.ACT_RELU, m, n, k, buf.data_ptr(), k + n + 8, w.data_ptr(), k, None, None, 0, buf.data_ptr() + 2 * k, k + n + 8, None, 0, None, 0))
    size = buf[:, :k].double().abs() @ w.double().abs().t()
    assert bool(((buf[:, k:k + n].double() - want).abs() <= 2.0 ** -11 * want + (k + 8) * F32 * size * 1.01 + 2.0 ** -25).all()) and bool((buf[:, k + n:] == tail).all())


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m", [1, 20, 600])
def test_not_finite_stays_in_its_row(hip, gated, m):
    """a NaN or an infinity in one sample reaches that sample's outputs alone"""
    layer = Layer(A.TYPE_HALF, A.ACT_RELU, m, 136, 80, gated=gated)
    layer.residual64 = None
    layer.x[1][m // 2, 3] = float("nan")
    y, pre = layer.forward()
    assert bool(y[1][m // 2].isnan().all()) and int(y[1].isnan().any(1).sum()) == 1
    layer.x[1][m // 2, 3] = float("inf")
    y, pre = layer.forward()
    assert not bool(pre[0][1][m // 2].isfinite().any()) and int((~pre[0][1].isfinite()).any(1).sum()) == 1
    dx = layer.backward(pre, "x")[0]
    assert int((~dx[1].isfinite()).any(1).sum()) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 512, 512), (3000, 136, 72), (12, 1024, 40)])
def test_same_bits_every_time(hip, gated, m, n, k):
    """no result depends on the order in which blocks run"""
    layer = Layer(A.TYPE_BFLOAT16, A.ACT_SILU, m, n, k, gated=gated)
    runs = []
    for _ in range(3):
        y, pre = layer.forward()
        dx, dw, db = layer.backward(pre)
        runs.append([v[1].clone() for v in [y, *pre, dx, *dw, *db]])
    for r in runs[1:]:
        assert all(bool((a == b).all()) for a, b in zip(r, runs[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_against_differences(hip, gated):
    """dx, dw, dbias against central differences of the loss sum(y * c) in 64 bits"""
    import torch
    layer = Layer(A.TYPE_HALF, A.ACT_SILU, 6, 10, 9, gated=gated)
    _, pre = layer.forward()
    # pre-activations that were rounded to half move the slopes by up to 2^-11 |z| (second derivative of silu <= 0.5), G once more, the result once more; differences with h = 2^-10 are
    # off by h^2 / 6 times the third derivative (< 0.4 |w|^3 |x|^3 ...): all together below 2^-7 of the sums of magnitudes
    dx, dw, db = layer.backward(pre)
    x, w, b, c = layer.x[1].double(), [v[1].double() for v in layer.w], [v[1].double() for v in layer.bias], layer.dy[1].double()

    def loss(x, w, b):
        z = [x @ v.t() + q for v, q in zip(w, b)]
        y = z[0] * torch.sigmoid(z[0])
        return float(((y * z[1] if gated else y) * c).sum())
    h = 2.0 ** -10
    for tensor, got in [(x, dx[1])] + [(v, d[1]) for v, d in zip(w, dw)] + [(q, d[1]) for q, d in zip(b, db)]:
        flat, grads = tensor.view(-1) if tensor.is_contiguous() else None, got.double().reshape(-1)
        assert flat is not None
        scale = float(grads.abs().max()) + 2.0 ** -6
        for i in range(0, flat.numel(), max(1, flat.numel() // 12)):
            old = float(flat[i])
            flat[i] = old + h; up = loss(x, w, b)
            flat[i] = old - h; down = loss(x, w, b)
            flat[i] = old
            assert abs((up - down) / (2 * h) - float(grads[i])) <= 2.0 ** -6 * scale


@pytest.mark.gpu
def test_other_stream_and_graph(hip):
    """the work is on the caller's stream; a captured forward + backward, replayed with new inputs, gives the eager results"""
    import torch
    for gated in (False, True):
        for m in (1, 3000):
            layer = Layer(A.TYPE_HALF, A.ACT_SILU, m, 136, 72, gated=gated)
            st = torch.cuda.Stream()
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                y, pre = layer.forward(stream=st.cuda_stream)
                grads = layer.backward(pre, stream=st.cuda_stream)
            st.synchronize()
            layer.residual64 = None
            layer.check_forward(y, pre)
            layer.check_backward(pre, *grads)
            L = lib()
            size = (L.ngp_gated_workspace_size if gated else L.ngp_linear_workspace_size)(m, 136, 72, 1)
            ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
            dx, dw, db = grads
            P = layer.p

            def step(s):
                if gated:
                    A.check(L, L.ngp_gated_forward(s, layer.type, layer.act, m, 136, 72, P(layer.x), 72, P(layer.w[0]), P(layer.w[1]), 72, P(layer.bias[0]), P(layer.bias[1]), P(y), 136, P(pre[0]), P(pre[1]), 136, None, 0))
                    A.check(L, L.ngp_gated_backward(s, layer.type, layer.act, m, 136, 72, P(layer.x), 72, P(layer.w[0]), P(layer.w[1]), 72, P(pre[0]), P(pre[1]), 136, P(layer.dy), 136, P(dx), 72, P(dw[0]), P(dw[1]), 72,
                                                    P(db[0]), P(db[1]), ws.data_ptr(), size))
                else:
                    A.check(L, L.ngp_linear_forward(s, layer.type, layer.act, m, 136, 72, P(layer.x), 72, P(layer.w[0]), 72, P(layer.bias[0]), None, 0, P(y), 136, P(pre[0]), 136, None, 0))
                    A.check(L, L.ngp_linear_backward(s, layer.type, layer.act, m, 136, 72, P(layer.x), 72, P(layer.w[0]), 72, P(pre[0]), 136, P(layer.dy), 136, P(dx), 72, P(dw[0]), 72, P(db[0]), ws.data_ptr(), size))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step(torch.cuda.current_stream().cuda_stream)
            for k in range(4):
                layer.x[1].copy_(torch.randn(m, 72, device="cuda") * (1 + k))
                graph.replay()
                torch.cuda.synchronize()
                got = [v[1].clone() for v in [y, *pre, dx, *dw, *db]]
                for v in [y, *pre, dx, *dw, *db]:
                    v[1].fill_(5.0)
                ws.fill_(255)
                step(None)
                torch.cuda.synchronize()
                for a, b in zip(got, [v[1] for v in [y, *pre, dx, *dw, *db]]):
                    assert bool((a == b).all())


@pytest.mark.gpu
def test_far_offsets(hip):
    """rows that lie further than 2^32 bytes into a buffer (a wide concatenation's columns)"""
    import torch
    L, m, n, k, stride = lib(), 70_000, 16, 24, 40_000
    buf = torch.zeros(m * stride // 2, dtype=torch.int32, device="cuda").view(torch.float16)[:m * stride].view(m, stride)  # 5.6 GB
    g = torch.Generator(device="cuda").manual_seed(3)
    buf[:, :k] = torch.randn(m, k, device="cuda", generator=g).half()
    w = (torch.randn(n, k, device="cuda", generator=g) / 8).half()
    A.check(L, L.ngp_linear_forward(None, A.TYPE_HALF, A.ACT_NONE, m, n, k, buf.data_ptr(), stride, w.data_ptr(), k, None, None, 0, buf.data_ptr() + 2 * 64, stride, None, 0, None, 0))
    x = buf[:, :k].double()
    want, size = x @ w.double().t(), x.abs() @ w.double().abs().t()
    assert bool(((buf[:, 64:64 + n].double() - want).abs() <= 2.0 ** -11 * want.abs() + (k + 8) * F32 * size * 1.01 + 2.0 ** -25).all())
    dy = buf[:, 64:64 + n]
    dw = torch.zeros(n, k, dtype=torch.float16, device="cuda")
    size_ws = L.ngp_linear_workspace_size(m, n, k, 1)
    ws = torch.empty(max(size_ws, 16), dtype=torch.uint8, device="cuda")
    dy.mul_(2.0 ** -8)
    A.check(L, L.ngp_linear_backward(None, A.TYPE_HALF, A.ACT_NONE, m, n, k, buf.data_ptr(), stride, w.data_ptr(), k, None, 0, dy.data_ptr(), stride, buf.data_ptr() + 2 * 128, stride, dw.data_ptr(), k, None, ws.data_ptr(), size_ws))
    d = dy.double()
    want, size = d @ w.double(), d.abs() @ w.double().abs()
    assert bool(((buf[:, 128:128 + k].double() - want).abs() <= 2.0 ** -11 * want.abs() + (n + 8) * F32 * size * 1.01 + 2.0 ** -25).all())
    want, size = d.t() @ x, d.t().abs() @ x.abs()
    assert bool(((dw.double() - want).abs() <= 2.0 ** -11 * want.abs() + (m + 8) * F32 * size * 1.01 + 2.0 ** -25).all())


@pytest.mark.gpu
def test_block_of_layers_with_the_trainer(hip):
    """As they are used together: frequency-encoded positions -> linear (relu) -> gated block with a residual -> linear to 3 colours; gradients through all of them against 64-bit autograd,
    the whole gradient clipped by its global norm, beside an encmlp model whose gradient vector is one of the tensors and whose optimizer step follows."""
    import torch
    L = lib()
    dev = "cuda"
    g = torch.Generator().manual_seed(5)
    m, k0, h, f = 1000, 63, 128, 192
    T = torch.float16
    pos = torch.rand(m, 3, generator=g)
    enc = torch.cat([pos] + [fn(pos * 2.0 ** i * math.pi) for i in range(10) for fn in (torch.sin, torch.cos)], 1)
    x0 = enc.to(T).to(dev)
    P = {n: (torch.randn(*s, generator=g) * math.sqrt(2.0 / (s[0] + s[-1]))).to(T).to(dev) for n, s in
         dict(w1=(h, k0), wg=(f, h), wu=(f, h), wd=(h, f), wo=(3, h)).items()}
    B = {n: (torch.randn(s, generator=g) * 0.1).to(T).to(dev) for n, s in dict(b1=h, bg=f, bu=f, bd=h, bo=3).items()}
    target = torch.rand(m, 3, generator=g).to(dev)
    e = lambda *s: torch.full(s, float("nan"), dtype=T, device=dev)
    z1, h1, zg, zu, hf, h2, y = e(m, h), e(m, h), e(m, f), e(m, f), e(m, f), e(m, h), e(m, 3)
    t = A.TYPE_HALF
    d = lambda v: v.data_ptr()
    A.check(L, L.ngp_linear_forward(None, t, A.ACT_RELU, m, h, k0, d(x0), k0, d(P["w1"]), k0, d(B["b1"]), None, 0, d(h1), h, d(z1), h, None, 0))
    A.check(L, L.ngp_gated_forward(None, t, A.ACT_SILU, m, f, h, d(h1), h, d(P["wg"]), d(P["wu"]), h, d(B["bg"]), d(B["bu"]), d(hf), f, d(zg), d(zu), f, None, 0))
    A.check(L, L.ngp_linear_forward(None, t, A.ACT_NONE, m, h, f, d(hf), f, d(P["wd"]), f, d(B["bd"]), d(h1), h, d(h2), h, None, 0, None, 0))
    A.check(L, L.ngp_linear_forward(None, t, A.ACT_NONE, m, 3, h, d(h2), h, d(P["wo"]), h, d(B["bo"]), None, 0, d(y), 3, None, 0, None, 0))
    scale = 128.0
    dy = ((y.float() - target) * (2 * scale / (3 * m))).to(T)
    G = {n: e(*v.shape) for n, v in {**P, **B}.items()}
    dh2, dhf, dh1, dx0, dh1b = e(m, h), e(m, f), e(m, h), e(m, k0), e(m, h)
    size = max(L.ngp_linear_workspace_size(m, n, k, 1) for n, k in ((h, k0), (h, f), (3, h)))
    size = max(size, L.ngp_gated_workspace_size(m, f, h, 1))
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    W = (d(ws), size)
    A.check(L, L.ngp_linear_backward(None, t, A.ACT_NONE, m, 3, h, d(h2), h, d(P["wo"]), h, None, 0, d(dy), 3, d(dh2), h, d(G["wo"]), h, d(G["bo"]), *W))
    A.check(L, L.ngp_linear_backward(None, t, A.ACT_NONE, m, h, f, d(hf), f, d(P["wd"]), f, None, 0, d(dh2), h, d(dhf), f, d(G["wd"]), f, d(G["bd"]), *W))
    A.check(L, L.ngp_gated_backward(None, t, A.ACT_SILU, m, f, h, d(h1), h, d(P["wg"]), d(P["wu"]), h, d(zg), d(zu), f, d(dhf), f, d(dh1b), h, d(G["wg"]), d(G["wu"]), h, d(G["bg"]), d(G["bu"]), *W))
    dh1 = dh1b + dh2
    A.check(L, L.ngp_linear_backward(None, t, A.ACT_RELU, m, h, k0, d(x0), k0, d(P["w1"]), k0, d(z1), h, d(dh1), h, d(dx0), k0, d(G["w1"]), k0, d(G["b1"]), *W))
    # 64-bit autograd of the same network from the same halfs
    Q = {n: v.double().requires_grad_(True) for n, v in {**P, **B}.items()}
    q0 = x0.double().requires_grad_(True)
    a1 = (q0 @ Q["w1"].t() + Q["b1"]).relu()
    gate = a1 @ Q["wg"].t() + Q["bg"]
    a2 = (gate * torch.sigmoid(gate) * (a1 @ Q["wu"].t() + Q["bu"])) @ Q["wd"].t() + Q["bd"] + a1
    out = a2 @ Q["wo"].t() + Q["bo"]
    assert float((y.double() - out).abs().max()) <= 2.0 ** -6 * float(out.abs().max())  # four layers of roundings of 2^-11, each of which the next two widen a few times
    (out * dy.double()).sum().backward()
    # every gradient passed at most five roundings of 2^-11 whose sums have random signs, against its own norm; relu units whose z rounds across zero (a share of 2^-10) change sides: 2^-5 = sqrt(2^-10)
    for n in G:
        ref = Q[n].grad
        assert float((G[n].double() - ref).norm()) <= 2.0 ** -5 * float(ref.norm()), n
    assert float((dx0.double() - q0.grad).norm()) <= 2.0 ** -5 * float(q0.grad.norm())
    # beside the image model's own gradient vector
    from common import dptr
    cfg = A.image_encmlp_config(log2_hashmap_size=15, image_resolution=256)
    em = C.c_void_p()
    A.check(L, L.ngp_encmlp_create(C.byref(cfg), 3, C.byref(em)))
    try:
        np_, nm = C.c_uint64(), C.c_uint64()
        L.ngp_encmlp_n_params(em, C.byref(np_), C.byref(nm))
        uv = torch.rand(4096, 2, generator=g).to(dev)
        tgt = torch.rand(4096, 3, generator=g).to(dev)
        grads = C.c_void_p()
        A.check(L, L.ngp_encmlp_param_ptrs(em, None, None, None, C.byref(grads)))
        A.check(L, L.ngp_encmlp_training_step(em, None, dptr(uv), 2, 4096, dptr(tgt), 3, A.LOSS_L2, C.c_float(scale), None, None, 0))
        torch.cuda.synchronize()
        names = sorted(G)
        table = (A.Gradient * (len(names) + 1))()
        for i, n in enumerate(names):
            table[i] = A.Gradient(d(G[n]), d(G[n]), G[n].numel(), A.TYPE_HALF, 0)
        table[len(names)] = A.Gradient(grads.value, grads.value, np_.value, A.TYPE_HALF, 0)
        before = {n: G[n].clone() for n in names}
        norm = torch.zeros(2, device=dev)
        cws = torch.empty(L.ngp_gradient_workspace_size(), dtype=torch.uint8, device=dev)
        A.check(L, L.ngp_gradient_norm(None, len(names), table, scale, d(norm), d(cws), cws.numel()))
        mine = math.sqrt(sum(float(before[n].double().square().sum()) for n in names)) / scale
        assert abs(float(norm[0]) - mine) <= 2.0 ** -22 * mine
        A.check(L, L.ngp_gradient_norm(None, len(names) + 1, table, scale, d(norm), d(cws), cws.numel()))
        whole = float(norm[0])
        assert whole > mine
        A.check(L, L.ngp_clip_gradients(None, len(names) + 1, table, scale, whole / 4, d(norm), d(cws), cws.numel()))
        for n in names:
            want = before[n].double() * 0.25
            assert bool(((G[n].double() - want).abs() <= 2.0 ** -11 * want.abs() * 1.001 + 2.0 ** -25).all())
        A.check(L, L.ngp_gradient_norm(None, len(names) + 1, table, scale, d(norm) + 4, d(cws), cws.numel()))
        assert abs(float(norm[1]) - whole / 4) <= 2.0 ** -10 * whole / 4
        A.check(L, L.ngp_encmlp_optimizer_step(em, None, C.c_float(scale)))
        torch.cuda.synchronize()
    finally:
        L.ngp_encmlp_destroy(em)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [A.TYPE_HALF, A.TYPE_BFLOAT16])
@pytest.mark.parametrize("m,n,k,gated", [(333, 777, 501, False), (257, 650, 321, True), (1000, 1000, 1003, False), (40, 2100, 1202, False), (3000, 263, 255, False)])
@pytest.mark.parametrize("pad,shift", [((0, 0, 0), 0), ((3, 2, 1), 1)])
def test_odd_lines(hip, type_, m, n, k, gated, pad, shift):
    """many products over lines that are no whole 16-byte pieces"""
    run_layer(Layer(type_, A.ACT_SILU, m, n, k, gated=gated, residual=not gated, pad=pad, shift=shift))


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [A.TYPE_HALF, A.TYPE_BFLOAT16])
@pytest.mark.parametrize("m,n,k,gated,act", [(160, 16, 3223, False, A.ACT_EXPONENTIAL), (1, 40, 500, True, A.ACT_SILU), (100, 16, 64, False, A.ACT_EXPONENTIAL), (37, 200, 136, True, A.ACT_GELU),
                                             (4, 8192, 500, False, A.ACT_RELU), (2000, 16, 8, False, A.ACT_LOGISTIC), (300, 33, 1000, True, A.ACT_NONE), (2, 129, 63, False, A.ACT_NONE)])
def test_few_gradients(hip, type_, m, n, k, gated, act):
    """small sets of gradients of the pre-activations are not rounded between the products: a value and what it lost leave u^2 of it (the lost part is rounded), and 2 u^2 covers that"""
    layer = Layer(type_, act, m, n, k, gated=gated, x_scale=0.5)
    layer.residual64 = None
    _, pre = layer.forward()
    layer.check_backward(pre, *layer.backward(pre), g_rounding=2 * U[type_] ** 2)
    layer.untouched()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(700, 777, 400), (300, 1001, 1000), (5000, 131, 264)])
@pytest.mark.parametrize("pad,shift", [((0, 0, 0), 0), ((0, 0, 5), 1)])
@pytest.mark.parametrize("want", ["xwb", "xw"])
def test_no_activation(hip, m, n, k, pad, shift, want):
    """the gradient of the outputs is that of the pre-activations, in whole pieces or not"""
    run_layer(Layer(A.TYPE_HALF, A.ACT_NONE, m, n, k, pad=pad, shift=shift), want=want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,gated,pad", [(263001, 256, 16, False, 0), (131073, 256, 24, False, 8), (263001, 128, 16, True, 0), (17001, 4099, 40, False, 0), (600001, 120, 400, False, 8)])
def test_outputs_beyond_the_caches(hip, m, n, k, gated, pad):
    run_layer(Layer(A.TYPE_HALF, A.ACT_RELU, m, n, k, gated=gated, residual=not gated, pad=(0, 0, pad)), backward=False)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,gated", [(1500, 504, 200, False), (700, 400, 512, True), (150, 1001, 1000, False)])
@pytest.mark.parametrize("pad,shift", [((5, 0, 5), 0), ((0, 3, 2), 0), ((2, 6, 4), 2), ((2, 4, 1), 1), ((0, 0, 0), 3)])
def test_whole_pieces_at_any_stride(hip, m, n, k, gated, pad, shift):
    """lines of whole 16-byte pieces that begin at even or odd elements, inputs and weights apart"""
    run_layer(Layer(A.TYPE_BFLOAT16, A.ACT_GELU, m, n, k, gated=gated, residual=not gated, pad=pad, shift=shift))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 16, 17, 32])
@pytest.mark.parametrize("n,k", [(8, 8192), (5, 4099), (40, 12290), (1000, 33), (2500, 129), (130, 1025)])
@pytest.mark.parametrize("gated,pad,shift", [(False, (0, 0, 0), 0), (True, (0, 0, 0), 0), (False, (1, 0, 1), 1), (True, (2, 4, 0), 2)])
def test_few_samples(hip, m, n, k, gated, pad, shift):
    """the sum shared by wavefronts and, where the outputs are few, by blocks"""
    run_layer(Layer(A.TYPE_HALF, A.ACT_GELU, m, n, k, gated=gated, residual=not gated, pad=pad, shift=shift), backward=False)
    run_layer(Layer(A.TYPE_BFLOAT16, A.ACT_SILU, m, n, k, gated=gated, residual=not gated, pad=pad, shift=shift), save=False, backward=False)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,gated", [(33, 8, 8, False), (33, 16, 256, False), (50, 9, 11, True), (1000, 100, 200, False), (777, 64, 40, True), (2049, 128, 129, False), (515, 33, 250, True), (4100, 250, 100, False),
                                         (33001, 256, 256, False), (32768, 255, 250, False), (33333, 128, 255, True), (40000, 200, 256, False), (100, 64, 512, False), (1000, 33, 257, False), (513, 31, 500, True), (33000, 128, 509, False),
                                         (32770, 64, 300, True)])
@pytest.mark.parametrize("pad,shift", [((0, 0, 0), 0), ((1, 3, 5), 1)])
def test_narrow_layers(hip, m, n, k, gated, pad, shift):
    """all weights in one compute unit, every size of it, samples that do not fill the last block"""
    run_layer(Layer(A.TYPE_HALF, A.ACT_SILU, m, n, k, gated=gated, residual=not gated, pad=pad, shift=shift))
    run_layer(Layer(A.TYPE_BFLOAT16, A.ACT_GELU, m, n, k, gated=gated, bias=False, pad=pad, shift=shift), want="xw")


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [A.TYPE_HALF, A.TYPE_BFLOAT16])
@pytest.mark.parametrize("m,n,k,gated", [(3700, 3593, 136, False), (3601, 1800, 72, True), (200, 96, 20000, False), (100, 40, 9001, True), (20000, 136, 264, True), (136, 264, 5008, False), (33, 4104, 1032, False), (4100, 4100, 40, False)])
def test_tiles(hip, type_, m, n, k, gated):
    """256 x 256 tiles with ragged edges; sums split over blocks in the forward pass, in dX, in dW; the two products of a backward pass side by side with either one the longer"""
    run_layer(Layer(type_, A.ACT_RELU, m, n, k, gated=gated, residual=not gated))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,gated", [(2, 16, 8192, False), (100, 48, 9000, True), (257, 650, 321, True), (40000, 64, 64, False)])
def test_bits_of_shared_sums(hip, m, n, k, gated):
    """sums that blocks share are joined in a fixed order, whatever the workspace held"""
    layer = Layer(A.TYPE_HALF, A.ACT_SILU, m, n, k, gated=gated)
    runs = []
    for _ in range(3):
        y, pre = layer.forward()
        dx, dw, db = layer.backward(pre)
        runs.append([v[1].clone() for v in [y, *pre, dx, *dw, *db]])
    for r in runs[1:]:
        assert all(bool((a == b).all()) for a, b in zip(r, runs[0]))
    layer.untouched()


@pytest.mark.gpu
def test_two_layers_at_once(hip):
    """two streams, and two graphs replayed on two streams, each layer with a workspace of its own"""
    import torch
    layers = [Layer(A.TYPE_HALF, A.ACT_SILU, m, n, k, gated=g, seed=i) for i, (m, n, k, g) in enumerate([(300, 264, 1001, False), (300, 264, 1001, True), (5, 24, 9000, False), (900, 136, 2048, False)])]
    L, want = lib(), []
    P = Layer.p

    def buffers(a):
        y, pre = a.out(a.m, a.n), [a.out(a.m, a.n) for _ in a.w]
        dx, dw, db = a.out(a.m, a.k), [a.out(a.n, a.k) for _ in a.w], [a.out(1, a.n) for _ in a.w]
        size = (L.ngp_gated_workspace_size if a.gated else L.ngp_linear_workspace_size)
        sizes = size(a.m, a.n, a.k, 0), size(a.m, a.n, a.k, 1)
        return y, pre, dx, dw, db, torch.full((max(sizes) + 16,), 255, dtype=torch.uint8, device="cuda"), sizes

    def run(a, b, s):
        y, pre, dx, dw, db, ws, sizes = b
        m, n, k = a.m, a.n, a.k
        if a.gated:
            A.check(L, L.ngp_gated_forward(s, a.type, a.act, m, n, k, P(a, a.x), k, P(a, a.w[0]), P(a, a.w[1]), k, P(a, a.bias[0]), P(a, a.bias[1]), P(a, y), n, P(a, pre[0]), P(a, pre[1]), n, ws.data_ptr(), sizes[0]))
            A.check(L, L.ngp_gated_backward(s, a.type, a.act, m, n, k, P(a, a.x), k, P(a, a.w[0]), P(a, a.w[1]), k, P(a, pre[0]), P(a, pre[1]), n, P(a, a.dy), n, P(a, dx), k, P(a, dw[0]), P(a, dw[1]), k,
                                            P(a, db[0]), P(a, db[1]), ws.data_ptr(), sizes[1]))
        else:
            A.check(L, L.ngp_linear_forward(s, a.type, a.act, m, n, k, P(a, a.x), k, P(a, a.w[0]), k, P(a, a.bias[0]), None, 0, P(a, y), n, P(a, pre[0]), n, ws.data_ptr(), sizes[0]))
            A.check(L, L.ngp_linear_backward(s, a.type, a.act, m, n, k, P(a, a.x), k, P(a, a.w[0]), k, P(a, pre[0]), n, P(a, a.dy), n, P(a, dx), k, P(a, dw[0]), k, P(a, db[0]), ws.data_ptr(), sizes[1]))

    def results(b):
        return [v[1].clone() for v in [b[0], *b[1], b[2], *b[3], *b[4]]]
    work = [buffers(a) for a in layers]
    for a, b in zip(layers, work):
        run(a, b, None)
        torch.cuda.synchronize()
        want.append(results(b))
        for v in [b[0], *b[1], b[2], *b[3], *b[4]]:
            v[1].fill_(3.0)
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    for _ in range(3):
        for a, b, st in zip(layers, work, streams):
            run(a, b, st.cuda_stream)
    torch.cuda.synchronize()
    for b, w in zip(work, want):
        assert all(bool((p == q).all()) for p, q in zip(results(b), w))
        for v in [b[0], *b[1], b[2], *b[3], *b[4]]:
            v[1].fill_(4.0)
    graphs = []
    for a, b in zip(layers, work):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(a, b, torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for b, w in zip(work, want):
            assert all(bool((p == q).all()) for p, q in zip(results(b), w))
            for v in [b[0], *b[1], b[2], *b[3], *b[4]]:
                v[1].fill_(5.0)
            b[5].fill_(255)
        torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ refusals (host only: nothing is launched)

def forward_args(**kw):
    a = dict(stream=None, type=A.TYPE_HALF, act=A.ACT_RELU, m=8, n=16, k=32, x=0x10000, xs=32, w=0x20000, ws=32, bias=0x30000, residual=None, rs=0, y=0x40000, ys=16, pre=0x50000, ps=16, work=None, size=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,what", [
    (dict(type=2), "type"), (dict(type=-1), "type"), (dict(act=6), "activation"), (dict(act=-1), "activation"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"),
    (dict(xs=31), "stride of x"), (dict(ws=31), "stride of w"), (dict(ys=15), "stride of y"), (dict(ps=15), "stride of pre"), (dict(residual=0x60000, rs=15), "stride of residual"),
    (dict(x=0x10001), "aligned"), (dict(bias=0x30001), "aligned"), (dict(y=0x10010), "y overlaps x"), (dict(y=0x20000), "y overlaps w"), (dict(pre=0x40000), "overlaps"), (dict(y=0x30000), "y overlaps bias"),
    (dict(residual=0x40010, rs=16), "y overlaps residual"), (dict(residual=0x40000, rs=17), "y overlaps residual"), (dict(m=1 << 31), "at most"), (dict(n=(1 << 24) + 1, ys=1 << 25, ps=1 << 25), "at most"),
    (dict(m=0x7fffffff, n=1 << 20, ys=1 << 20, pre=None), "tiles"), (dict(xs=1 << 50), "too large"), (dict(m=1 << 20, xs=1 << 39), "stride of x too large"), (dict(m=1 << 20, ys=1 << 30), "stride of y too large")])
def test_forward_refusals(kw, what):
    L = lib()
    assert L.ngp_linear_forward(*forward_args(**kw)) != 0
    assert what in L.ngp_last_error().decode()


def backward_args(**kw):
    a = dict(stream=None, type=A.TYPE_HALF, act=A.ACT_RELU, m=8, n=16, k=32, x=0x10000, xs=32, w=0x20000, ws=32, pre=0x30000, ps=16, dy=0x40000, dys=16, dx=0x50000, dxs=32, dw=0x60000, dws=32, dbias=0x70000,
             work=0x80000, size=1 << 20)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,what", [
    (dict(pre=None), "pre-activations"), (dict(dy=None), "null"), (dict(x=None), "dw without x"), (dict(w=None), "dx without w"), (dict(size=16), "workspace"), (dict(work=None), "workspace"), (dict(work=0x80008), "workspace"),
    (dict(dx=0x60000), "overlaps"), (dict(dx=0x10000), "overlaps"), (dict(dw=0x20000), "overlaps"), (dict(dx=0x40000), "overlaps"), (dict(work=0x40000), "overlaps"), (dict(dbias=0x60010), "overlaps"),
    (dict(dxs=31), "stride of dx"), (dict(dws=31), "stride of dw"), (dict(type=3), "type")])
def test_backward_refusals(kw, what):
    L = lib()
    assert L.ngp_linear_backward(*backward_args(**kw)) != 0
    assert what in L.ngp_last_error().decode()


def gated_args(**kw):
    a = dict(stream=None, type=A.TYPE_HALF, act=A.ACT_SILU, m=8, n=16, k=32, x=0x10000, xs=32, wg=0x20000, wu=0x21000, ws=32, bg=None, bu=None, y=0x40000, ys=16, gp=0x50000, up=0x51000, ps=16, work=None, size=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,what", [(dict(wu=None), "null"), (dict(y=0x21000), "overlaps"), (dict(up=0x50000), "overlaps"), (dict(act=9), "activation"), (dict(ps=3), "stride"), (dict(bu=0x3), "aligned")])
def test_gated_refusals(kw, what):
    L = lib()
    assert L.ngp_gated_forward(*gated_args(**kw)) != 0
    assert what in L.ngp_last_error().decode()


@pytest.mark.parametrize("kw,what", [(dict(dwu=None), "together"), (dict(up=None), "null"), (dict(wg=None), "dx without"), (dict(x=None), "dw without"), (dict(size=64), "workspace"), (dict(dbu=0x60000), "overlaps")])
def test_gated_backward_refusals(kw, what):
    L = lib()
    a = dict(stream=None, type=A.TYPE_HALF, act=A.ACT_SILU, m=8, n=16, k=32, x=0x10000, xs=32, wg=0x20000, wu=0x21000, ws=32, gp=0x30000, up=0x31000, ps=16, dy=0x40000, dys=16, dx=0x50000, dxs=32, dwg=0x60000, dwu=0x61000,
             dws=32, dbg=0x70000, dbu=0x71000, work=0x80000, size=1 << 20)
    a.update(kw)
    assert L.ngp_gated_backward(*a.values()) != 0
    assert what in L.ngp_last_error().decode()


def test_arguments_in_order_ask_for_a_device():
    """the same calls with nothing wrong get as far as the device"""
    L = lib()
    if L.ngp_device_available():
        pytest.skip("has a GPU: these addresses are not its own")
    for f, a in ((L.ngp_linear_forward, forward_args()), (L.ngp_linear_forward, forward_args(residual=0x40000, rs=16)), (L.ngp_linear_backward, backward_args()), (L.ngp_gated_forward, gated_args()),
                 (L.ngp_linear_forward, forward_args(x=0x10000, xs=64, y=0x10040, ys=64, pre=None))):  # (last: columns 0..31 and 32..47 of one buffer)
        assert f(*a) != 0 and "no HIP device" in L.ngp_last_error().decode()


def test_workspace_sizes():
    L = lib()
    for m, n, k in ((1, 1, 1), (0, 8, 8), (262144, 256, 256), (8192, 8192, 2048), (1 << 20, 64, 64)):
        for f, problems in ((L.ngp_linear_workspace_size, 1), (L.ngp_gated_workspace_size, 2)):
            assert f(m, n, k, 0) >= 0
            s = f(m, n, k, 1)
            # at most the gradients of the pre-activations and a bounded set of partial sums; layers whose weights fit a compute unit never store the former, the others have to
            assert s <= problems * 2 * m * (n + 8) + (300 << 20) and (s >= problems * 2 * m * n or (problems * n <= 256 and k <= 256))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(2, 16, 8192), (100, 64, 9000), (1000, 1000, 1003)])
def test_forward_workspace(gated, m, n, k):
    """sums that blocks share and padded operands need room in the forward pass too: its size is asked for and held to"""
    L = lib()
    size = (L.ngp_gated_workspace_size if gated else L.ngp_linear_workspace_size)(m, n, k, 0)
    assert size > 0
    a = [1 << 32 | i << 28 for i in range(8)]
    for work, have, what in ((None, 0, "workspace"), (a[6], size - 1, "workspace"), (a[6] + 8, size, "workspace"), (a[3], size, "overlaps"), (a[0], size, "overlaps")):
        if gated:
            rc = L.ngp_gated_forward(None, A.TYPE_HALF, A.ACT_SILU, m, n, k, a[0], k, a[1], a[2], k, None, None, a[3], n, a[4], a[5], n, work, have)
        else:
            rc = L.ngp_linear_forward(None, A.TYPE_HALF, A.ACT_SILU, m, n, k, a[0], k, a[1], k, None, None, 0, a[3], n, a[4], n, work, have)
        assert rc != 0 and what in L.ngp_last_error().decode()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(512, 768, 8500001), (512, 1000, (1 << 24) - 1), (1000, 2000, (1 << 21) + 1), (128, 64, 1 << 24), (70000, 800, (1 << 21) + 8)])
def test_no_copies_of_very_long_lines(gated, m, n, k):
    """the tiles that read copied operands reach a tile's lines by 31-bit offsets (255 lines of 2^21 elements): longer lines are not copied, so no size asks for room for them"""
    L = lib()
    size = L.ngp_gated_workspace_size if gated else L.ngp_linear_workspace_size
    cols = (2 if gated else 1) * n
    copies = 2 * (m + cols) * (k // 8 * 8)
    partial = 600 << 20  # two sets of partial sums of at most 256 MB and a little, and G
    assert size(m, n, k, 0) < min(copies, partial) + 2 * cols * m and size(m, n, k, 1) < min(copies, partial) + 4 * cols * (m + 8)
    k = 1 << 21  # the longest that are (the backward pass has the room for lines at odd strides)
    assert size(2000, 1000, k, 1) >= 2 * (2000 + (2000 if gated else 1000)) * k and size(2000, 1000, k - 1, 0) >= 2 * (2000 + (2000 if gated else 1000)) * k


def test_sizes_out_of_range_are_answered():
    """a size may be asked for before anything is checked: every value has an answer, and the call itself refuses what is out of range.  (In a process of its own: a rule that never ends is to fail.)"""
    import os
    import subprocess
    import sys
    code = """
import itertools, ngp_abi as A
L, big = A.load_hip(), 0xffffffff
for m, n, k, back in itertools.product((0, 5, big), (0, 3, big), (0, 7, 1 << 31, big), (0, 1)):
    L.ngp_linear_workspace_size(m, n, k, back), L.ngp_gated_workspace_size(m, n, k, back)
assert L.ngp_linear_workspace_size(5, 0, big, 0) == 0 and L.ngp_gated_workspace_size(5, 0, 1 << 31, 0) == 0
for n, k in ((0, big), (0, 1 << 31), (big, big)):
    assert L.ngp_linear_forward(None, A.TYPE_HALF, A.ACT_RELU, 5, n, k, 0x1000, k, 0x2000, k, None, None, 0, 0x3000, n, None, 0, 1 << 32, 1 << 60) != 0
    assert 'at most' in L.ngp_last_error().decode(), L.ngp_last_error()
print('answered')
"""
    path = os.pathsep.join([os.path.dirname(os.path.abspath(A.__file__)), os.environ.get("PYTHONPATH", "")])
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": path}, capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "answered" in r.stdout, r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,gated", [(34001, 770, 4001, False), (17001, 390, 8003, True)])
def test_long_copies(hip, m, n, k, gated):
    """more 16-byte pieces than the copying launch has threads"""
    run_layer(Layer(A.TYPE_HALF, A.ACT_RELU, m, n, k, gated=gated))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,gated,want", [(700, 777, 501, False, "x"), (700, 777, 501, False, "w"), (600, 400, 333, True, "x"), (600, 400, 333, True, "w"), (700, 777, 501, False, "xw")])
def test_copies_of_what_is_read(hip, m, n, k, gated, want):
    """dX alone reads the weights and dW alone the inputs: the other operand's copy is not made (as much of the workspace is written with it as without), and the results are those of the whole call"""
    import torch
    layer = Layer(A.TYPE_HALF, A.ACT_SILU, m, n, k, gated=gated)
    _, pre = layer.forward()
    parts = layer.backward(pre, want)
    written = int((layer.ws != 255).sum())
    x, w = layer.x, layer.w
    if want == "x":
        layer.x = None
    elif want == "w":
        layer.w = [None for _ in w]
    without = layer.backward(pre, want)
    assert written == int((layer.ws != 255).sum())
    layer.x, layer.w = x, w
    whole = layer.backward(pre)
    for a, b, c in zip([parts[0], *parts[1]], [without[0], *without[1]], [whole[0], *whole[1]]):
        assert (a is None and b is None) or (torch.equal(a[1], b[1]) and torch.equal(a[1], c[1]))
    layer.untouched()



@pytest.mark.gpu
@pytest.mark.parametrize("type_,most", [(A.TYPE_HALF, 16.0), (A.TYPE_BFLOAT16, 60.0)])
@pytest.mark.parametrize("m,n", [(1, 64), (40, 64), (3000, 64), (3000, 520)])
@pytest.mark.parametrize("gated", [False, True])
def test_logistic_slope_in_both_tails(hip, type_, most, m, n, gated):
    """p (1 - p) keeps its bits far from zero, on either side.  The weights are the unit matrix, so dX is G itself: a 16-bit rounding (u) and 32-bit operations, of which the exponential's are off by
    its argument times 2^-24 twice (log2 e and the product with it are rounded) and a few steps, the other ones by one or two each: (2 |z| + 16) 2^-24."""
    import torch
    layer = Layer(type_, A.ACT_LOGISTIC, m, n, n, gated=gated, bias=False)
    g = torch.Generator().manual_seed(m + n)
    pre = [layer.matrix((torch.rand(m, n, generator=g) * 2 - 1) * most, 0)] + [layer.matrix(torch.randn(m, n, generator=g), 0) for _ in layer.w[1:]]
    layer.dy[1].copy_((2.0 ** 12 * (1 + torch.rand(m, n, generator=g))).to(layer.dtype).cuda())
    z, dy = pre[0][1].double(), layer.dy[1].double()
    p, q = torch.sigmoid(z), torch.sigmoid(-z)
    for which, want in enumerate([dy * p * q * (pre[1][1].double() if gated else 1)] + ([dy * p] if gated else [])):
        for i, w in enumerate(layer.w):
            w[1].copy_(torch.eye(n, device="cuda") * (i == which))
        dx = layer.backward(pre, "x")[0]
        tol = (U[type_] + 1.01 * (2 * z.abs() + 16) * F32) * want.abs() + TINY[type_]
        off = (dx[1].double() - want).abs() / tol
        assert bool((off <= 1).all()), f"{float(off.max()):.2f} of the tolerance at z = {float(z.reshape(-1)[off.argmax()]):.2f}"
    layer.untouched()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [A.TYPE_HALF, A.TYPE_BFLOAT16])
@pytest.mark.parametrize("m,n,k", [(3700, 3593, 136), (300, 264, 512), (100, 48, 9000), (5, 16, 8192), (20, 100, 200), (300, 200, 333), (100, 48, 9001), (1000, 1000, 1003), (263001, 256, 16), (1000001, 72, 24), (700003, 100, 17),
                                   (5000, 64, 64)])
@pytest.mark.parametrize("pad", [0, 5])
def test_residual_in_place_every_way(hip, type_, m, n, k, pad):
    """large and small tiles, shared sums, few rows with and without, tiles through registers, copied operands, narrow layers with and without the exchange between neighbouring samples"""
    layer = Layer(type_, A.ACT_GELU, m, n, k, residual=True, pad=(0, 0, pad))
    layer.residual64 = layer.residual[1].double().clone()
    y, pre = layer.forward(save=m < 100000, y_is_residual=True)
    layer.check_forward(y, pre)
    layer.untouched()
    y[1].fill_(float("nan"))
    assert bool(y[0].isnan().all()), "written beside y"


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [A.TYPE_HALF, A.TYPE_BFLOAT16])
@pytest.mark.parametrize("m,n,k,gated", [(3000, 64, 72, True), (2001, 30, 255, True), (33000, 128, 256, True), (3000, 64, 72, False), (5001, 16, 250, False), (33000, 250, 256, False)])
def test_parts_of_the_gradient_of_narrow_layers(hip, type_, m, n, k, gated):
    """each output alone is bit for bit the one of the whole call, and no operand that it does not need is looked at"""
    layer = Layer(type_, A.ACT_SILU, m, n, k, gated=gated)
    layer.residual64 = None
    _, pre = layer.forward()
    whole = layer.backward(pre)
    layer.check_backward(pre, *whole)
    x, w = layer.x, layer.w
    for want, pick in (("x", lambda r: [r[0]]), ("w", lambda r: r[1]), ("b", lambda r: r[2]), ("xb", lambda r: [r[0], *r[2]]), ("wb", lambda r: [*r[1], *r[2]])):
        layer.x = x if "w" in want else None
        layer.w = w if "x" in want else [None for _ in w]
        part = layer.backward(pre, want)
        for a, b in zip(pick(part), pick(whole)):
            assert bool((a[1] == b[1]).all())
    layer.untouched()


@pytest.mark.gpu
@pytest.mark.parametrize("stride", [1 << 21, (1 << 21) + 2, (1 << 21) + 8])
@pytest.mark.parametrize("m,n,k,gated", [(130, 264, 64, False), (130, 136, 64, True), (90, 64, 64, False), (257, 130, 72, False), (5, 40, 64, True)])
def test_far_lines(hip, stride, m, n, k, gated):
    """lines either side of what a tile's 31-bit offsets allow (2^21 elements from line to line)"""
    run_layer(Layer(A.TYPE_HALF, A.ACT_SILU, m, n, k, gated=gated, residual=not gated, pad=(stride - k, stride - k, stride - n)))


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(2, 16, 8192), (100, 64, 9000), (100, 64, 9001), (1000, 1000, 1003), (17, 40, 12290), (600, 400, 1003)])
def test_behind_the_forward_workspace(hip, gated, m, n, k):
    layer = Layer(A.TYPE_HALF, A.ACT_SILU, m, n, k, gated=gated)
    layer.residual64 = None
    layer.check_forward(*layer.forward())
    size = (lib().ngp_gated_workspace_size if gated else lib().ngp_linear_workspace_size)(m, n, k, 0)
    assert layer.ws.numel() == size + 64 and bool((layer.ws[size:] == 255).all())


@pytest.mark.parametrize("gated", [False, True])
def test_forward_workspace_sizes(gated):
    """nothing where one launch does it all; room for partial sums, at most 256 MB of them, and for the operands' padded copies elsewhere"""
    L = lib()
    size = L.ngp_gated_workspace_size if gated else L.ngp_linear_workspace_size
    cols = 2 if gated else 1
    for m, n, k in ((1, 1, 1), (0, 8, 8), (8, 0, 8), (8, 8, 0), (1, 8192, 2048), (262144, 256 // cols, 256), (65521, 256 // cols, 63), (8192, 8192, 2048), (1 << 20, 64, 64)):
        assert size(m, n, k, 0) == 0, (m, n, k)
    for m, n, k in ((2, 16, 8192), (32, 100, 10000), (100, 64, 9000), (64, 200, 100000)):
        assert 0 < size(m, n, k, 0) <= 256 << 20, (m, n, k)
    for m, n, k in ((1000, 1000, 1003), (65536, 1032, 1004)):
        copies = 2 * (m + cols * n) * ((k + 7) // 8 * 8)
        assert copies <= size(m, n, k, 0) <= copies + (256 << 20), (m, n, k)
