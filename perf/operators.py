"""Cases of the dense-layer operators: ngp_linear_* (matrix product with bias, activation and residual), ngp_gated_*
(gated feed-forward projections) and ngp_clip_gradients (global gradient norm and clipping), with their plain forms.

A matrix is row-major; weights are [outputs][inputs] like the framework's own MLP layers."""
import math
import os
import random
import sys

import numpy as np
import torch

own = False  # True: the framework's kernels; False: elementary torch operations in 32 bits

TYPES = {"half": torch.float16, "bfloat16": torch.bfloat16, "float": torch.float32}
CODES = {"half": 0, "bfloat16": 1, "float": 2}                                                      # NGP_TYPE_*
ACTS = {"none": 0, "relu": 1, "logistic": 2, "exponential": 3, "silu": 4, "gelu": 5}                # NGP_ACT_*


def listed():
    return [
        # one query (a pixel, a token) through a wide layer with a residual connection: latency
        dict(name="linear one row", op="linear", backward=False, type="half", act="gelu", m=1, k=2048, n=2048, bias=True, residual=True, save=False, pad=0),
        # the first layer of a frequency-encoded radiance field (3 + 3 * 2 * 10 inputs) over a ray batch of odd size, training: rows start at odd addresses
        dict(name="linear 63 inputs", op="linear", backward=False, type="half", act="relu", m=65521, k=63, n=256, bias=True, residual=False, save=True, pad=0),
        # a wide residual layer over a full batch: the largest forward product
        dict(name="linear wide", op="linear", backward=False, type="bfloat16", act="gelu", m=8192, k=4096, n=4096, bias=True, residual=True, save=True, pad=0),
        # backward of a 256-neuron hidden layer over the trainer's 2^18 samples: a long sum for the weights, memory bound
        dict(name="linear backward samples", op="linear", backward=True, type="half", act="relu", m=262144, k=256, n=256, bias=True, residual=False, save=False, pad=0),
        # backward of a layer with ragged sizes
        dict(name="linear backward ragged", op="linear", backward=True, type="bfloat16", act="silu", m=5003, k=1000, n=777, bias=True, residual=False, save=False, pad=0),
        # one query through a gated block
        dict(name="gated one row", op="gated", backward=False, type="bfloat16", act="silu", m=1, k=2048, n=8192, bias=False, residual=False, save=False, pad=0),
        # a gated block over an ordinary batch, training (both pre-activations are kept)
        dict(name="gated batch", op="gated", backward=False, type="half", act="silu", m=4096, k=1024, n=4096, bias=False, residual=False, save=True, pad=0),
        # its gradients on a large batch: the most work of all
        dict(name="gated backward", op="gated", backward=True, type="bfloat16", act="silu", m=8192, k=2048, n=8192, bias=False, residual=False, save=False, pad=0),
        # the same with odd sizes and biases
        dict(name="gated backward ragged", op="gated", backward=True, type="half", act="gelu", m=777, k=500, n=1333, bias=True, residual=False, save=False, pad=12),
        # the matrices of the image model's MLP
        dict(name="clip mlp", op="clip", types="half", tensors=3, elements=7168, over=True, loss_scale=128.0),
        # a NeRF model's hash grid and matrices in half, its per-image latents and cameras in float
        dict(name="clip nerf", op="clip", types="mixed", tensors=9, elements=12206480, over=True, loss_scale=128.0),
        # many tensors of a wide network, fine as they are
        dict(name="clip many", op="clip", types="bfloat16", tensors=300, elements=400_000_003, over=True, loss_scale=1.0),
    ]


def _size(rng, low, high):
    """Spread over the logarithm; odd ones and multiples of 8 both come up."""
    v = max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))
    return v if rng.random() < 0.5 else max(low, min(high, -(-v // 8) * 8))


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(["linear", "linear", "gated", "gated", "clip"])
        if op == "clip":
            c = dict(op=op, types=rng.choice(["half", "bfloat16", "float", "mixed"]), tensors=int(round(math.exp(rng.uniform(0.0, math.log(300.0))))),
                     elements=_size(rng, 5000, 400_000_003), over=rng.random() < 0.7, loss_scale=rng.choice([1.0, 128.0]))
        else:
            c = dict(op=op, backward=rng.random() < 0.5, type=rng.choice(["half", "bfloat16"]), act=rng.choice(list(ACTS)), m=_size(rng, 1, 262144), k=_size(rng, 16, 8192),
                     n=_size(rng, 16, 8192), bias=rng.random() < 0.6, residual=op == "linear" and rng.random() < 0.5, save=rng.random() < 0.5, pad=rng.choice([0, 0, 0, 8, 5]))
            if c["backward"]:
                c["residual"] = c["save"] = False
        w = work(c)
        if all(w[k] <= most[k] for k in most):
            return c


def _tensor_sizes(case):
    """Ragged sizes that add up to case["elements"]: a few large tensors, many small ones."""
    n, r = case["tensors"], random.Random(case["tensors"] * 1000003 + case["elements"])
    share = [math.exp(2.5 * r.gauss(0.0, 1.0)) for _ in range(n)]
    rest = case["elements"] - n
    sizes = [1 + int(rest * s / sum(share)) for s in share]
    sizes[sizes.index(max(sizes))] += case["elements"] - sum(sizes)
    return sizes


def _tensor_types(case):
    if case["types"] != "mixed":
        return [case["types"]] * case["tensors"]
    sizes = _tensor_sizes(case)
    small = sorted(range(len(sizes)), key=lambda i: sizes[i])[:len(sizes) // 3]  # the small ones in float: latents, cameras
    return ["float" if i in small else "half" for i in range(len(sizes))]


def work(case):
    if case["op"] == "clip":
        size = {"half": 2, "bfloat16": 2, "float": 4}
        return {"bytes": 2 * sum(s * size[t] for s, t in zip(_tensor_sizes(case), _tensor_types(case))) + 4, "flops": 3 * case["elements"]}
    m, n, k, back = case["m"], case["n"], case["k"], case["backward"]
    proj = 2 if case["op"] == "gated" else 1
    values = m * k + proj * n * k + m * n + (proj * n if case["bias"] else 0)
    if back:  # x, w, the pre-activations, dy -> dx, dw, dbias
        values += m * k + proj * n * k + (proj * n if case["bias"] else 0) + (proj * m * n if proj == 2 or case["act"] != "none" else 0)
    else:
        values += (m * n if case["residual"] else 0) + (proj * m * n if case["save"] else 0)
    return {"bytes": 2 * values, "flops": (4 if back else 2) * proj * m * n * k}


def _matrix(g, rows, cols, dtype, scale, pad=0, positive=False):
    """`pad` more columns behind each row: the matrix is then a part of a wider buffer."""
    v = torch.randn(rows, cols + pad, generator=g, device="cuda") * scale
    return (v.abs() if positive else v).to(dtype)[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case=case)
    if case["op"] == "clip":
        sizes, types = _tensor_sizes(case), _tensor_types(case)
        s["grads"], s["clipped"], place = {}, {}, {t: 0 for t in TYPES}
        for t in sorted(set(types)):
            n = sum(z for z, u in zip(sizes, types) if u == t)
            v = torch.randn(n, generator=g, device="cuda")
            v *= torch.rand(n, generator=g, device="cuda") > 0.4       # cells that no sample of the batch touched
            s["grads"][t] = (v * (0.05 if t != "float" else 0.5)).to(TYPES[t])
            s["clipped"][t] = torch.zeros_like(s["grads"][t])
        table = np.zeros(len(sizes), dtype=[("grad", "<u8"), ("clipped", "<u8"), ("size", "<u8"), ("type", "<i4"), ("reserved", "<i4")])  # struct ngp_gradient
        table["size"], table["type"] = sizes, [CODES[t] for t in types]
        at = []
        for z, t in zip(sizes, types):
            at.append(place[t])
            place[t] += z * s["grads"][t].element_size()
        table["grad"] = [s["grads"][t].data_ptr() + a for t, a in zip(types, at)]
        table["clipped"] = [s["clipped"][t].data_ptr() + a for t, a in zip(types, at)]
        norm = math.sqrt(sum(float(v.double().square().sum()) for v in s["grads"].values())) / case["loss_scale"]
        s["max_norm"] = float(np.float32(norm * (0.37 if case["over"] else 1.9)))
        s["table"], s["norm"] = table, torch.zeros(1, device="cuda")
        return s
    dtype, m, n, k = TYPES[case["type"]], case["m"], case["n"], case["k"]
    xavier = math.sqrt(2.0 / (n + k))
    s["x"] = _matrix(g, m, k, dtype, 1.0, case["pad"], positive=case["act"] == "relu")
    names = ["w_gate", "w_up"] if case["op"] == "gated" else ["w"]
    for name in names:
        s[name] = _matrix(g, n, k, dtype, xavier)
        s["bias" + name[1:]] = _matrix(g, 1, n, dtype, 0.3)[0] if case["bias"] else None
    if not case["backward"]:
        s["residual"] = _matrix(g, m, n, dtype, 1.0) if case["residual"] else None
        s["y"] = torch.zeros(m, n, dtype=dtype, device="cuda")
        for name in names:
            s["pre" + name[1:]] = torch.zeros(m, n, dtype=dtype, device="cuda") if case["save"] else None
        return s
    s["dy"] = _matrix(g, m, n, dtype, 2.0 ** -4, case["pad"])
    for name in names:  # the forward pass's pre-activations
        z = s["x"].float() @ s[name].float().t()
        s["pre" + name[1:]] = (z if s["bias" + name[1:]] is None else z + s["bias" + name[1:]].float()).to(dtype)
        del z
        s["d" + name] = torch.zeros(n, k, dtype=dtype, device="cuda")
        s["dbias" + name[1:]] = torch.zeros(n, dtype=dtype, device="cuda") if case["bias"] else None
    s["dx"] = torch.zeros(m, k, dtype=dtype, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------- plain forms

def _act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return z.clamp_min(0.0)
    if name == "logistic":
        return 1.0 / (1.0 + torch.exp(-z))
    if name == "exponential":
        return torch.exp(z)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))


def _act_derivative(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).float()
    if name == "exponential":
        return torch.exp(z)
    if name in ("logistic", "silu"):
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 - p) if name == "logistic" else p * (1.0 + z * (1.0 - p))
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _project(x, w, bias):
    z = x @ w.float().t()
    return z if bias is None else z + bias.float()


def _plain(s):
    case = s["case"]
    if case["op"] == "clip":
        norm = torch.sqrt(sum(v.double().square().sum() for v in s["grads"].values())) / case["loss_scale"]
        scale = (s["max_norm"] / norm).clamp(max=1.0).float()
        return {"clipped": {t: (v.float() * scale).to(v.dtype) for t, v in s["grads"].items()}, "norm": norm.float().reshape(1)}
    dtype, act, x = TYPES[case["type"]], case["act"], s["x"].float()
    if case["op"] == "linear" and not case["backward"]:
        z = _project(x, s["w"], s["bias"])
        y = _act(act, z)
        y = y if s["residual"] is None else y + s["residual"].float()
        return {"y": y.to(dtype), "pre": z.to(dtype) if case["save"] else None}
    if case["op"] == "linear":
        g = s["dy"].float() * _act_derivative(act, s["pre"].float())
        return {"dx": (g @ s["w"].float()).to(dtype), "dw": (g.t() @ x).to(dtype), "dbias": g.sum(0).to(dtype) if case["bias"] else None}
    if not case["backward"]:
        gate, up = _project(x, s["w_gate"], s["bias_gate"]), _project(x, s["w_up"], s["bias_up"])
        return {"y": (_act(act, gate) * up).to(dtype), "pre_gate": gate.to(dtype) if case["save"] else None, "pre_up": up.to(dtype) if case["save"] else None}
    dy, gate = s["dy"].float(), s["pre_gate"].float()
    gg = dy * s["pre_up"].float() * _act_derivative(act, gate)
    gu = dy * _act(act, gate)
    return {"dx": (gg @ s["w_gate"].float() + gu @ s["w_up"].float()).to(dtype), "dw_gate": (gg.t() @ x).to(dtype), "dw_up": (gu.t() @ x).to(dtype),
            "dbias_gate": gg.sum(0).to(dtype) if case["bias"] else None, "dbias_up": gu.sum(0).to(dtype) if case["bias"] else None}


# ---------------------------------------------------------------------------------------------- the framework's calls

def _library():
    path = os.path.join(os.getcwd(), "instant-ngp_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ngp_abi
    return ngp_abi


def _p(t):
    return None if t is None else t.data_ptr()


def _workspace(s, size):
    if "workspace" not in s:
        s["workspace"] = torch.empty(max(int(size()), 16), dtype=torch.uint8, device="cuda")
    return s["workspace"].data_ptr(), s["workspace"].numel()


def _own(s):
    A, case = _library(), s["case"]
    lib = A.load_hip()
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "clip":
        ws = _workspace(s, lib.ngp_gradient_workspace_size)
        A.check(lib, lib.ngp_clip_gradients(stream, len(s["table"]), s["table"].ctypes.data, case["loss_scale"], s["max_norm"], s["norm"].data_ptr(), *ws))
        return {"clipped": s["clipped"], "norm": s["norm"]}
    head = (CODES[case["type"]], ACTS[case["act"]], case["m"], case["n"], case["k"])
    x, xs = s["x"].data_ptr(), s["x"].stride(0)
    n, k = case["n"], case["k"]
    if case["op"] == "linear" and not case["backward"]:
        ws = _workspace(s, lambda: lib.ngp_linear_workspace_size(case["m"], n, k, 0))
        A.check(lib, lib.ngp_linear_forward(stream, *head, x, xs, s["w"].data_ptr(), k, _p(s["bias"]), _p(s["residual"]), n, s["y"].data_ptr(), n, _p(s["pre"]), n, *ws))
        return {"y": s["y"], "pre": s["pre"]}
    if case["op"] == "linear":
        ws = _workspace(s, lambda: lib.ngp_linear_workspace_size(case["m"], n, k, 1))
        A.check(lib, lib.ngp_linear_backward(stream, *head, x, xs, s["w"].data_ptr(), k, s["pre"].data_ptr(), n, s["dy"].data_ptr(), s["dy"].stride(0),
                                             s["dx"].data_ptr(), k, s["dw"].data_ptr(), k, _p(s["dbias"]), *ws))
        return {"dx": s["dx"], "dw": s["dw"], "dbias": s["dbias"]}
    weights = (s["w_gate"].data_ptr(), s["w_up"].data_ptr(), k)
    if not case["backward"]:
        ws = _workspace(s, lambda: lib.ngp_gated_workspace_size(case["m"], n, k, 0))
        A.check(lib, lib.ngp_gated_forward(stream, *head, x, xs, *weights, _p(s["bias_gate"]), _p(s["bias_up"]), s["y"].data_ptr(), n, _p(s["pre_gate"]), _p(s["pre_up"]), n, *ws))
        return {"y": s["y"], "pre_gate": s["pre_gate"], "pre_up": s["pre_up"]}
    ws = _workspace(s, lambda: lib.ngp_gated_workspace_size(case["m"], n, k, 1))
    A.check(lib, lib.ngp_gated_backward(stream, *head, x, xs, *weights, s["pre_gate"].data_ptr(), s["pre_up"].data_ptr(), n, s["dy"].data_ptr(), s["dy"].stride(0),
                                        s["dx"].data_ptr(), k, s["dw_gate"].data_ptr(), s["dw_up"].data_ptr(), k, _p(s["dbias_gate"]), _p(s["dbias_up"]), *ws))
    return {"dx": s["dx"], "dw_gate": s["dw_gate"], "dw_up": s["dw_up"], "dbias_gate": s["dbias_gate"], "dbias_up": s["dbias_up"]}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------- 64 bits

def _value64(act, z):
    """(act(z), act'(z)) in 64 bits."""
    one = torch.ones_like(z)
    if act == "none":
        return z, one
    if act == "relu":
        return torch.where(z > 0, z, 0 * one), torch.where(z > 0, one, 0 * one)
    if act == "exponential":
        return z.exp(), z.exp()
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z.square() / 2) / math.sqrt(2.0 * math.pi)
    p, q = torch.sigmoid(z), torch.sigmoid(-z)
    return (p, p * q) if act == "logistic" else (z * p, p + z * p * q)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        wide = {t: v.to(torch.float64) for t, v in s["grads"].items()}
        norm = math.sqrt(math.fsum(float(torch.dot(v, v)) for v in wide.values())) / case["loss_scale"]
        c = s["max_norm"] / norm if norm > s["max_norm"] else 1.0
        return {"clipped": {t: v.mul_(c) for t, v in wide.items()}, "norm": torch.tensor([norm], dtype=torch.float64)}
    x, act = s["x"].double(), case["act"]
    names = ["_gate", "_up"] if case["op"] == "gated" else [""]
    w = [s["w" + e].double() for e in names]
    if not case["backward"]:
        z = [torch.mm(x, v.t()) for v in w]
        if case["bias"]:
            z = [v.add_(s["bias" + e].double()) for v, e in zip(z, names)]
        y = _value64(act, z[0])[0]
        y = y * z[1] if case["op"] == "gated" else y + s["residual"].double() if case["residual"] else y
        return {"y": y, **{"pre" + e: v if case["save"] else None for v, e in zip(z, names)}}
    value, slope = _value64(act, s["pre" + names[0]].double())
    dy = s["dy"].double()
    g = [dy * slope] if case["op"] == "linear" else [dy * slope * s["pre_up"].double(), dy * value]
    out = {"dx": sum(torch.mm(a, b) for a, b in zip(g, w))}
    for a, e in zip(g, names):
        out["dw" + e] = torch.mm(x.t(), a).t()
        out["dbias" + e] = torch.mv(a.t(), torch.ones(len(a), dtype=torch.float64, device=a.device)) if case["bias"] else None
    return out
