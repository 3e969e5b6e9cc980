"""The operators around a linear layer's weight, as they are measured: what each one reads, writes and
computes, in plain torch and through this repository's entry points.

  orthogonalize   O = NS(G): a few Newton-Schulz steps bring a matrix's singular values near 1.
                  X0 = G / (|G|_F + eps);  X <- a X + (b A + c A A) X with A = X X^T (X^T X on the right
                  where G has more rows than columns).
  muon_update     one optimiser step of a weight matrix: M <- mu M + G; U = G + mu M (or M without the
                  look-ahead); W <- (1 - lr wd) W - lr scale NS(U).  W and M are updated in place.
  w4_quantize     a [k, n] weight in 4 bits: groups of `group` consecutive k of one output column share a
                  scale (symmetric: code - 8 times max|w| / 7; otherwise (code - zero) times range / 15).
  w4_dequantize   the [k, n] fp32 values that such a weight stands for.
  matmul_w4       y = [relu](x W + bias) for a few rows x, W read in 4 bits.

Layout of a 4-bit weight: packed[n][kw] 32-bit words, kw = ceil(k / group) * group / 8, eight consecutive k
of one column in a word, code 2p of the eight in bits 4p..4p+3 and code 2p+1 in bits 16+4p..16+4p+3;
scales[n][ceil(k / group)] fp32; zeros of the same shape, bytes, or none for the symmetric form.
"""
import math

import torch

own = False

COEF = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
NIBBLE = (0, 16, 4, 20, 8, 24, 12, 28)   # bit position of code i of a word


# ---- the cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # the classifier head of the small network (784-128-10): one launch's latency is all there is
        dict(name="ortho 128x10", op="orthogonalize", rows=128, cols=10, steps=5),
        # its hidden layer
        dict(name="ortho 784x128", op="orthogonalize", rows=784, cols=128, steps=5),
        # a hidden layer of the wide network (784-4096-4096-4096-10): the largest product chain
        dict(name="ortho 4096x4096", op="orthogonalize", rows=4096, cols=4096, steps=5),
        # odd sizes, momentum without the look-ahead, no decay, as a user's own layer has them
        dict(name="muon 333x1001", op="muon_update", rows=333, cols=1001, steps=5, nesterov=False, decay=0.0),
        # the wide network's first layer: a short side that fills few tiles
        dict(name="muon 784x4096", op="muon_update", rows=784, cols=4096, steps=5, nesterov=True, decay=0.01),
        # its hidden layers: the step that decides the training time
        dict(name="muon 4096x4096", op="muon_update", rows=4096, cols=4096, steps=5, nesterov=True, decay=0.01),
        # a hidden layer quantised once training is done, and the values it stands for then, to see what was lost
        dict(name="quantize 4096x4096 g128", op="w4_quantize", k=4096, n=4096, group=128, symmetric=True),
        # the same of a large layer with zero points, both extents ragged
        dict(name="quantize 8191x10007 g32 z", op="w4_quantize", k=8191, n=10007, group=32, symmetric=False),
        # one sample through the hidden layer: bound by the weight's bytes
        dict(name="w4 1x4096x4096 g128", op="matmul_w4", m=1, k=4096, n=4096, group=128, symmetric=True, bias=True, relu=True),
        # a few samples through a small odd layer: latency
        dict(name="w4 3x1001x517 g32 z", op="matmul_w4", m=3, k=1001, n=517, group=32, symmetric=False, bias=True, relu=False),
        # a few samples through a layer larger than the L2 cache
        dict(name="w4 4x16384x16384 g64 z", op="matmul_w4", m=4, k=16384, n=16384, group=64, symmetric=False, bias=False, relu=False),
        # a batch of the small network's size through the hidden layer: bound by arithmetic
        dict(name="w4 64x4096x4096 g128", op="matmul_w4", m=64, k=4096, n=4096, group=128, symmetric=True, bias=True, relu=True),
    ]


def _size(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, v | rng.randint(0, 1)))     # odd more often than not


def draw(rng):
    op = rng.choice(["orthogonalize", "muon_update", "w4_quantize", "matmul_w4", "matmul_w4"])
    if op == "orthogonalize":
        return dict(op=op, rows=_size(rng, 8, 4096), cols=_size(rng, 8, 4096), steps=rng.choice([3, 5, 5]))
    if op == "muon_update":
        return dict(op=op, rows=_size(rng, 8, 4096), cols=_size(rng, 8, 4096), steps=5, nesterov=rng.random() < 0.7,
                    decay=rng.choice([0.0, 0.01]))
    if op == "w4_quantize":
        return dict(op=op, k=_size(rng, 32, 8192), n=_size(rng, 8, 10000), group=rng.choice([32, 64, 128]), symmetric=rng.random() < 0.5)
    return dict(op=op, m=_size(rng, 1, 64), k=_size(rng, 32, 16384), n=_size(rng, 8, 16384), group=rng.choice([32, 64, 128]),
                symmetric=rng.random() < 0.5, bias=rng.random() < 0.7, relu=rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------------
def _gradient(rows, cols, gen):
    """A weight gradient x^T d of a layer behind a ReLU: noise over inputs and units of different strength,
    plus the rank-one part that the inputs' positive mean adds."""
    dev = "cuda"
    g = torch.randn(rows, cols, device=dev, generator=gen)
    r = torch.exp(0.5 * torch.randn(rows, 1, device=dev, generator=gen))
    c = torch.exp(0.5 * torch.randn(1, cols, device=dev, generator=gen))
    mean = torch.randn(1, cols, device=dev, generator=gen)
    return (1e-3 * r * c * (g + mean)).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case)
    if op in ("orthogonalize", "muon_update"):
        rows, cols = case["rows"], case["cols"]
        s["g"] = _gradient(rows, cols, gen)
        if op == "orthogonalize":
            s["out"] = torch.empty_like(s["g"])
        else:
            s["w"] = torch.randn(rows, cols, device="cuda", generator=gen) / math.sqrt(rows)
            s["m"] = 3.0 * _gradient(rows, cols, gen)
            s["scale"] = math.sqrt(max(1.0, cols / rows))
    else:
        k, n, group = case["k"], case["n"], case["group"]
        groups = -(-k // group)
        if op == "w4_quantize":
            s["w"] = torch.randn(k, n, device="cuda", generator=gen) / math.sqrt(k)
            s["packed"] = torch.empty(n, groups * group // 8, device="cuda", dtype=torch.int32)
            s["scales"] = torch.empty(n, groups, device="cuda")
            s["zeros"] = None if case["symmetric"] else torch.empty(n, groups, device="cuda", dtype=torch.uint8)
            s["values"] = torch.empty(k, n, device="cuda")
        else:
            s["x"] = torch.relu(torch.randn(case["m"], k, device="cuda", generator=gen))       # a hidden activation
            s["scales"] = torch.rand(n, groups, device="cuda", generator=gen).add_(0.5).mul_(0.3 / math.sqrt(k))
            s["zeros"] = None if case["symmetric"] else torch.randint(6, 10, (n, groups), device="cuda", dtype=torch.uint8, generator=gen)
            zero = 8 if case["symmetric"] else s["zeros"].to(torch.int32).repeat_interleave(group // 8, dim=1)
            s["packed"] = torch.zeros(n, groups * group // 8, device="cuda", dtype=torch.int32)
            for at in NIBBLE:       # codes of weights that are normal around zero
                q = (2.5 * torch.randn(s["packed"].shape, device="cuda", generator=gen)).round_().to(torch.int32)
                s["packed"] |= (q + zero).clamp_(1 if case["symmetric"] else 0, 15) << at
            s["bias"] = 0.1 * torch.randn(n, device="cuda", generator=gen) if case["bias"] else None
            s["out"] = torch.empty(case["m"], n, device="cuda")
    if own:
        # what a user of the framework holds: its arrays (here over the same memory) and a 4-bit weight's handle
        import ctorch_b200 as cb
        import numpy as np

        def arr(t, dtype=np.float32):
            return None if not isinstance(t, torch.Tensor) else cb.DeviceArray(tuple(t.shape), dtype, _ptr=t.data_ptr(), _owner=t)

        s["dev"] = {key: arr(s.get(key)) for key in ("g", "out", "w", "m", "x", "bias", "values")}
        if "packed" in s:
            s["dev"]["w4"] = cb.ops.W4Weight(arr(s["packed"], np.uint32), arr(s["scales"]), arr(s["zeros"], np.uint8), k=k, n=n, group=group)
    return s


# ---- one pass ----------------------------------------------------------------------------------------
def _newton_schulz(g, steps, eps):
    tall = g.shape[0] > g.shape[1]
    a, b, c = COEF
    x = g / (g.square().sum().sqrt() + eps)
    for _ in range(steps):
        if tall:
            gram = x.T @ x
            x = a * x + x @ (b * gram + c * (gram @ gram))
        else:
            gram = x @ x.T
            x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x


def _codes(packed):
    """int codes [n, 8 kw] of the packed words."""
    at = torch.tensor(NIBBLE, device=packed.device, dtype=torch.int32)
    return ((packed[:, :, None] >> at) & 15).reshape(packed.shape[0], -1)


def _values(codes, scales, zeros, group, dtype=torch.float32):
    """Dequantised [n, groups * group]."""
    n = codes.shape[0]
    q = codes.reshape(n, -1, group).to(dtype)
    q = q - (8.0 if zeros is None else zeros.to(dtype)[:, :, None])
    return (q * scales.to(dtype)[:, :, None]).reshape(n, -1)


def _grouped(w, group):
    """[k, n] -> [n, groups, group], zero-padded along k."""
    k, n = w.shape
    pad = -k % group
    return torch.nn.functional.pad(w.T, (0, pad)).reshape(n, (k + pad) // group, group)


def _quantize(w, group, symmetric):
    """codes [n, groups, group] (int32), scales, zeros or None.  Scales are the nearest fp32 values;
    the quotients next to a rounding border are decided in 64 bits, ties to even."""
    v = _grouped(w, group)
    if symmetric:
        scales = (v.abs().amax(-1).double() / 7.0).float()
        zeros = None
        lo = torch.full_like(scales, 8.0, dtype=torch.float64)
    else:
        top, bottom = v.amax(-1).clamp(min=0.0), v.amin(-1).clamp(max=0.0)
        scales = ((top.double() - bottom.double()) / 15.0).float()
        lo = torch.where(scales > 0, torch.round(-bottom.double() / scales.double()), torch.zeros_like(scales, dtype=torch.float64))
        zeros = lo.to(torch.uint8)
    q = torch.where(scales[:, :, None] > 0, torch.round(v.double() / scales.double()[:, :, None]), torch.zeros_like(v, dtype=torch.float64))
    return (q + lo[:, :, None]).clamp(1.0 if symmetric else 0.0, 15.0).to(torch.int32), scales, zeros


def _pack(codes):
    """[n, groups, group] int32 codes -> [n, kw] int32 words."""
    c = codes.reshape(codes.shape[0], -1, 8)
    at = torch.tensor(NIBBLE, device=codes.device, dtype=torch.int32)
    return (c << at).sum(-1, dtype=torch.int32)


def _run_plain(s):
    op = s["op"]
    if op == "orthogonalize":
        return _newton_schulz(s["g"], s["steps"], EPS)
    if op == "muon_update":
        g, w, m = s["g"], s["w"], s["m"]
        m.mul_(0.95).add_(g)
        u = g + 0.95 * m if s["nesterov"] else m
        o = _newton_schulz(u, s["steps"], EPS)
        w.mul_(1.0 - 0.02 * s["decay"]).sub_(0.02 * s["scale"] * o)
        return w, m
    if op == "w4_quantize":
        codes, scales, zeros = _quantize(s["w"], s["group"], s["symmetric"])
        s["packed"].copy_(_pack(codes))
        s["scales"].copy_(scales)
        if zeros is not None:
            s["zeros"].copy_(zeros)
        s["values"].copy_(_values(_codes(s["packed"]), scales, zeros, s["group"])[:, :s["k"]].T)
        return [s["values"], s["scales"]] + ([] if zeros is None else [s["zeros"]])
    k = s["k"]
    w = _values(_codes(s["packed"]), s["scales"], s["zeros"], s["group"])[:, :k]
    y = s["x"] @ w.T
    if s["bias"] is not None:
        y = y + s["bias"]
    return torch.relu(y) if s["relu"] else y


def _run_own(s):
    import ctorch_b200 as cb
    op, d = s["op"], s["dev"]
    if op == "orthogonalize":
        cb.ops.orthogonalize(d["g"], steps=s["steps"], eps=EPS, out=d["out"])
        return s["out"]
    if op == "muon_update":
        cb.ops.muon_update(d["w"], d["g"], d["m"], lr=0.02, momentum=0.95, nesterov=s["nesterov"], weight_decay=s["decay"], scale=s["scale"],
                           steps=s["steps"], eps=EPS)
        return s["w"], s["m"]
    if op == "w4_quantize":
        cb.ops.w4_quantize(d["w"], group=s["group"], symmetric=s["symmetric"], out=d["w4"])
        cb.ops.w4_dequantize(d["w4"], out=d["values"])
        return [s["values"], s["scales"]] + ([] if s["zeros"] is None else [s["zeros"]])
    cb.ops.matmul_w4(d["x"], d["w4"], bias=d["bias"], relu=s["relu"], out=d["out"])
    return s["out"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op in ("orthogonalize", "muon_update"):
        size = case["rows"] * case["cols"]
        d, length = sorted((case["rows"], case["cols"]))
        # per step: one triangle of the Gram matrix, one of its square, the product with X
        flops = case["steps"] * (d * (d + 1) * length + d * (d + 1) * d + 2 * d * d * length)
        return dict(bytes=4 * size * (2 if op == "orthogonalize" else 5), flops=flops)
    groups = -(-case["k"] // case["group"])
    held = case["n"] * groups * (case["group"] // 2 + 4 + (0 if case["symmetric"] else 1))
    if op == "w4_quantize":
        return dict(bytes=8 * case["k"] * case["n"] + held, flops=5 * case["k"] * case["n"])
    m, k, n = case["m"], case["k"], case["n"]
    return dict(bytes=held + 4 * (m * k + m * n + (n if case["bias"] else 0)), flops=2 * m * k * n)


# ---- the definition, in 64 bits ----------------------------------------------------------------------
def _polar64(u, steps):
    """The same iteration on the Gram side: the step's polynomial in S = X X^T is applied as an operator."""
    flip = u.shape[0] > u.shape[1]
    x = u.t() if flip else u
    x = x / (torch.linalg.matrix_norm(x) + EPS)
    eye = torch.eye(x.shape[0], dtype=x.dtype, device=x.device)
    for _ in range(steps):
        s = torch.matmul(x, x.mT)
        x = torch.matmul(COEF[0] * eye + s @ (COEF[1] * eye + COEF[2] * s), x)
    return x.t() if flip else x


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "orthogonalize":
        return _polar64(s["g"].double(), case["steps"])
    if op == "muon_update":
        m = 0.95 * s["m"].double() + s["g"].double()
        u = s["g"].double() + 0.95 * m if case["nesterov"] else m
        return (1.0 - 0.02 * case["decay"]) * s["w"].double() - 0.02 * s["scale"] * _polar64(u, case["steps"]), m
    k, n, group = case["k"], case["n"], case["group"]
    groups = -(-k // group)
    if op == "w4_quantize":
        w = torch.zeros(groups * group, n, dtype=torch.float64, device="cuda")
        w[:k] = s["w"]
        w = w.reshape(groups, group, n)
        if case["symmetric"]:
            scale = w.abs().max(dim=1).values / 7
            least, most, zero = -7.0, 7.0, 0.0
        else:
            bottom = w.min(dim=1).values.clamp(max=0)
            scale = (w.max(dim=1).values.clamp(min=0) - bottom) / 15
            zero = (-bottom / scale.float().double()).nan_to_num(nan=0.0).round()
            least, most = (0 - zero)[:, None], (15 - zero)[:, None]
        scale = scale.float().double()[:, None]     # a scale is the nearest fp32 number: the codes are counted in it
        code = (w / scale).nan_to_num(nan=0.0).round()
        code = torch.minimum(torch.maximum(code, torch.as_tensor(least, device="cuda")), torch.as_tensor(most, device="cuda"))
        values = (code * scale).reshape(groups * group, n)[:k]
        return [values, scale[:, 0].t().contiguous()] + ([] if case["symmetric"] else [None])
    y = torch.zeros(case["m"], n, dtype=torch.float64, device="cuda")
    x = torch.zeros(case["m"], groups * group, dtype=torch.float64, device="cuda")
    x[:, :k] = s["x"]
    zero = 8.0 if s["zeros"] is None else None
    for i, at in enumerate(NIBBLE):     # code i of every word, all words at once
        q = ((s["packed"] >> at) & 15).double()                       # [n, kw]
        per = group // 8
        z = zero if zero is not None else s["zeros"].double().repeat_interleave(per, dim=1)
        y += x[:, i::8] @ ((q - z) * s["scales"].double().repeat_interleave(per, dim=1)).t()
    if s["bias"] is not None:
        y += s["bias"].double()
    return y.clamp(min=0) if case["relu"] else y
