"""Performance cases of the feed-forward operators: `nn.LayerNorm`, `nn.FusedLinear` and `nn.GroupedLinear`.

    listed()            the cases timed by name
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what the program holds before the call
    run(state)          one pass and its outputs: by the framework's modules where `own` is true, else in plain torch operations
    exact(case, seed)   the outputs from the definitions in 64 bits
    work(case)          bytes and floating-point operations the pass cannot do without

Three operators (`case["op"]`):

    norm      rows of `size` values, normalised, times a weight plus a bias
    linear    activation(x w^T + b), plus a residual where the case has one
    experts   the same product where the rows of each group have weights of their own; `tokens` rows sorted by group

`way`: "forward" (serving: nothing is kept for a backward pass), "backward" (the gradients, from what a forward pass has kept) or "step"
(a training forward and backward).  Values are FP32, as all of the framework's tensors are.  A step through "relu" is not among the
cases: its gradient turns on or off where a sum lies within its rounding of zero, whichever way the sum is computed."""
import math

import numpy as np
import torch

own = False

EPS = 1e-5


def listed():
    return [
        # the norm in front of one token's block: latency alone
        {"name": "norm_forward_token", "op": "norm", "way": "forward", "rows": 1, "size": 4096},
        # training, wide rows: HBM bandwidth, and a weight gradient summed over many rows
        {"name": "norm_backward_wide", "op": "norm", "way": "backward", "rows": 16384, "size": 4096},
        # an image's planes behind the last convolution (256 of 13 x 13) as one row: few long rows
        {"name": "norm_step_planes", "op": "norm", "way": "step", "rows": 200, "size": 43264},
        # short rows whose length no 16-byte access divides
        {"name": "norm_step_ragged", "op": "norm", "way": "step", "rows": 30011, "size": 333},
        # a classifier's first fully connected layer for one image: the weights' bytes
        {"name": "linear_forward_one", "op": "linear", "way": "forward", "rows": 1, "inputs": 9216, "outputs": 4096, "act": "relu",
         "residual": False},
        # a prompt or an evaluation batch through the widening product
        {"name": "linear_forward_large", "op": "linear", "way": "forward", "rows": 8192, "inputs": 4096, "outputs": 8192, "act": "gelu",
         "residual": False},
        # a training step through a square layer with a skip connection
        {"name": "linear_step_residual", "op": "linear", "way": "step", "rows": 2048, "inputs": 4096, "outputs": 4096, "act": "gelu",
         "residual": True},
        # gradients at sizes that no tile and no 16-byte access divides
        {"name": "linear_backward_ragged", "op": "linear", "way": "backward", "rows": 777, "inputs": 1531, "outputs": 1001, "act": "relu",
         "residual": False},
        # decoding a small batch: most experts get no row, the others one or two
        {"name": "experts_forward_few", "op": "experts", "way": "forward", "tokens": 24, "groups": 64, "inputs": 1024, "outputs": 2048,
         "act": "silu", "skew": 0.5, "routing": 1},
        # a prompt through a routed layer, loads uneven
        {"name": "experts_forward_prompt", "op": "experts", "way": "forward", "tokens": 8192, "groups": 16, "inputs": 1024, "outputs": 4096,
         "act": "gelu", "skew": 0.7, "routing": 2},
        # a training step through eight experts
        {"name": "experts_step", "op": "experts", "way": "step", "tokens": 6000, "groups": 8, "inputs": 2048, "outputs": 1408, "act": "silu",
         "skew": 0.3, "routing": 3},
        # many small groups, some empty, of odd sizes
        {"name": "experts_backward_ragged", "op": "experts", "way": "backward", "tokens": 1537, "groups": 37, "inputs": 333, "outputs": 515,
         "act": "none", "skew": 1.5, "routing": 4},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["norm", "linear", "experts"])
        way = rng.choice(["forward", "backward", "step"])
        if op == "norm":
            case = {"op": op, "way": way, "rows": _log(rng, 1, 32768), "size": _log(rng, 1, 65536)}
            if case["rows"] * case["size"] > 1 << 26:
                continue
            return case
        act = rng.choice(["none", "gelu", "silu"] if way == "step" else ["none", "relu", "gelu", "silu"])
        if op == "linear":
            case = {"op": op, "way": way, "rows": _log(rng, 1, 8192), "inputs": _log(rng, 16, 9216), "outputs": _log(rng, 8, 8192), "act": act,
                    "residual": rng.random() < 0.4}
        else:
            case = {"op": op, "way": way, "tokens": _log(rng, 1, 16384), "groups": _log(rng, 2, 128), "inputs": _log(rng, 16, 4096),
                    "outputs": _log(rng, 16, 4096), "act": act, "skew": round(rng.uniform(0.0, 1.5), 2), "routing": rng.randrange(1000)}
        w = work(case)
        if w["flops"] <= 5e11 and w["bytes"] <= 2e9:
            return case


def counts_of(case):
    """Rows of each group, as a router leaves them: a few groups get most (`skew`), some get none."""
    r = np.random.RandomState(case["routing"])
    p = r.permutation(np.arange(1.0, case["groups"] + 1.0) ** -case["skew"])
    return r.multinomial(case["tokens"], p / p.sum()).astype(np.int64)


# ------------------------------------------------------------------ inputs
class _State:
    def __init__(self, case):
        self.case = case


def _inputs(case, seed):
    """Everything the pass reads, drawn on the device from the seed."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    t = {}
    if case["op"] == "norm":
        rows, size = case["rows"], case["size"]
        # a residual stream: rows of different sizes around a mean of their own, some channels larger than the others
        channel = 1.0 + 4.0 * (torch.rand(size, device="cuda", generator=g) < 0.02)
        t["x"] = normal(rows, size) * channel * (0.5 + normal(rows, 1).abs()) + 0.3 * normal(rows, 1)
        t["weight"], t["bias"] = 1.0 + 0.1 * normal(size), 0.1 * normal(size)
        shape = (rows, size)
    else:
        i, o = case["inputs"], case["outputs"]
        lead = (case["groups"],) if case["op"] == "experts" else ()
        rows = case["tokens"] if case["op"] == "experts" else case["rows"]
        stdv = 1.0 / math.sqrt(i)
        t["x"] = normal(rows, i)
        t["weight"] = (torch.rand(lead + (o, i), device="cuda", generator=g) * 2 - 1) * (math.sqrt(3.0) * stdv)
        t["bias"] = 0.1 * normal(*lead, o)
        if case.get("residual"):
            t["residual"] = normal(rows, o)
        shape = (rows, o)
    if case["way"] != "forward":
        t["gradOutput"] = normal(*shape)
    if case["way"] == "backward":      # what the forward pass has kept
        if case["op"] == "norm":
            mean = t["x"].mean(1)
            t["mean"], t["invStd"] = mean, (t["x"] - mean[:, None]).square().mean(1).add(EPS).rsqrt()
        else:
            t["preactivation"] = normal(*shape)
    return t


def prepare(case, seed):
    s = _State(case)
    s.t = _inputs(case, seed)
    if case["op"] == "experts":
        s.counts = counts_of(case)
    if own:
        _modules(s)
    torch.cuda.synchronize()
    return s


class _Zeros:
    """Stands in for the host generator while a module is built: its parameters are the case's."""

    def uniform(self, shape, a, b):
        return np.zeros(shape, np.float32)


def _wrap(gt, t):
    """A torch.GPUTensor over a (contiguous) torch tensor's memory."""
    L = gt.lib()
    st = L.THGPUStorage_newWithData(t.data_ptr(), t.numel())
    v = gt.GPUTensor(_ptr=L.THGPUTensor_newWithStorage1d(st, 0, t.numel(), 1)).view(*t.shape)
    L.THGPUStorage_free(st)
    return v


def _modules(s):
    """The module of the case over the case's tensors, with its results in memory that torch sees too."""
    import mcw_cppamp_torch_b200 as gt
    c, t = s.case, s.t
    g = {k: _wrap(gt, v) for k, v in t.items()}
    if c["op"] == "norm":
        m = gt.nn.LayerNorm(c["size"], eps=EPS)
        rows, outputs = c["rows"], c["size"]
        t.setdefault("mean", torch.empty(rows, device="cuda"))
        t.setdefault("invStd", torch.empty(rows, device="cuda"))
        m.mean, m.invStd = _wrap(gt, t["mean"]), _wrap(gt, t["invStd"])
        s.input = g["x"]
    elif c["op"] == "linear":
        m = gt.nn.FusedLinear(c["inputs"], c["outputs"], c["act"], rng=_Zeros())
        rows, outputs = c["rows"], c["outputs"]
        s.input = [g["x"], g["residual"]] if c["residual"] else g["x"]
    else:
        m = gt.nn.GroupedLinear(c["groups"], c["inputs"], c["outputs"], c["act"], rng=_Zeros())
        rows, outputs = c["tokens"], c["outputs"]
        s.input = [g["x"], s.counts]
    if c["way"] == "forward":
        m.evaluate()
    else:
        s.gradOutput = g["gradOutput"]
        if "preactivation" in g:
            m.preactivation = g["preactivation"]
    m.weight, m.bias = g["weight"], g["bias"]
    for name, shape in (("gradWeight", t["weight"].shape), ("gradBias", t["bias"].shape), ("output", (rows, outputs)),
                        ("gradInput", t["x"].shape)):
        t[name] = torch.zeros(shape, device="cuda")
        setattr(m, name, _wrap(gt, t[name]))
    s.module = m
    gt.synchronize()


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    return {"norm": _plain_norm, "linear": _plain_linear, "experts": _plain_experts}[s.case["op"]](s.case, s.t, s)


GRADIENTS = ("gradInput", "gradWeight", "gradBias")


def _run_own(s):
    m, way = s.module, s.case["way"]
    if way != "backward":
        m.forward(s.input)
    if way != "forward":
        m.zeroGradParameters()
        m.backward(s.input, s.gradOutput)
    names = {"forward": ("output",), "backward": GRADIENTS, "step": ("output",) + GRADIENTS}[way]
    return {k: s.t[k] for k in names}


def _activation(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain_norm(c, t, s):
    x, way, out = t["x"], c["way"], {}
    if way == "backward":
        mean, inv = t["mean"][:, None], t["invStd"][:, None]
        xh = (x - mean) * inv
    else:
        mean = x.mean(1, keepdim=True)
        d = x - mean
        inv = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
        xh = d * inv
        out["output"] = xh * t["weight"] + t["bias"]
    if way != "forward":
        go = t["gradOutput"]
        gw = go * t["weight"]
        out["gradInput"] = inv * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
        out["gradWeight"], out["gradBias"] = (go * xh).sum(0), go.sum(0)
    return out


def _plain_linear(c, t, s):
    x, w, way, out = t["x"], t["weight"], c["way"], {}
    if way == "backward":
        z = t["preactivation"]
    else:
        z = x @ w.t() + t["bias"]
        out["output"] = _activation(z, c["act"]) + t["residual"] if c["residual"] else _activation(z, c["act"])
    if way != "forward":
        gz = t["gradOutput"] * _slope(z, c["act"])
        out["gradInput"], out["gradWeight"], out["gradBias"] = gz @ w, gz.t() @ x, gz.sum(0)
    return out


def _plain_experts(c, t, s):
    w, way, out, counts = t["weight"], c["way"], {}, s.counts.tolist()
    xs = t["x"].split(counts)
    if way == "backward":
        z = t["preactivation"]
    else:
        z = torch.cat([x @ wg.t() + b for x, wg, b in zip(xs, w, t["bias"])])
        out["output"] = _activation(z, c["act"])
    if way != "forward":
        gzs = (t["gradOutput"] * _slope(z, c["act"])).split(counts)
        out["gradInput"] = torch.cat([gz @ wg for gz, wg in zip(gzs, w)])
        out["gradWeight"] = torch.stack([gz.t() @ x for gz, x in zip(gzs, xs)])
        out["gradBias"] = torch.stack([gz.sum(0) for gz in gzs])
    return out


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    t = {k: v.double() for k, v in _inputs(case, seed).items()}
    x, way, out = t["x"], case["way"], {}
    if case["op"] == "norm":
        n = case["size"]
        mean = x.sum(1) / n
        variance = torch.einsum("ij,ij->i", x - mean[:, None], x - mean[:, None]) / n
        inv = (variance + EPS) ** -0.5
        if way == "backward":
            mean, inv = t["mean"], t["invStd"]
        unit = torch.einsum("ij,i->ij", x - mean[:, None], inv)
        if way != "backward":
            out["output"] = torch.addcmul(t["bias"], unit, t["weight"])
        if way != "forward":
            go = t["gradOutput"]
            one, two = torch.einsum("ij,j->i", go, t["weight"]) / n, torch.einsum("ij,j,ij->i", go, t["weight"], unit) / n
            out["gradInput"] = torch.einsum("ij,i->ij", go * t["weight"] - one[:, None] - two[:, None] * unit, inv)
            out["gradWeight"], out["gradBias"] = torch.einsum("ij,ij->j", go, unit), torch.einsum("ij->j", go)
        return out
    groups = case.get("groups", 1)
    weight, bias = t["weight"].reshape(groups, *t["weight"].shape[-2:]), t["bias"].reshape(groups, -1)
    counts = counts_of(case).tolist() if case["op"] == "experts" else [case["rows"]]
    ends = np.cumsum([0] + counts)
    part = [slice(int(a), int(b)) for a, b in zip(ends[:-1], ends[1:])]
    z = t.get("preactivation")
    if z is None:
        z = torch.cat([torch.einsum("ri,oi->ro", x[p], weight[g]) + bias[g] for g, p in enumerate(part)])
    normal_below = 0.5 * torch.erfc(-z / math.sqrt(2.0))         # of the standard normal distribution
    sigmoid = torch.where(z < 0, torch.exp(torch.clamp(z, max=0.0)), torch.ones_like(z)) / (1.0 + torch.exp(-z.abs()))
    if way != "backward":
        y = {"none": z, "relu": torch.clamp(z, min=0.0), "gelu": z * normal_below, "silu": z * sigmoid}[case["act"]]
        out["output"] = y + t["residual"] if case.get("residual") else y
    if way != "forward":
        slope = {"none": torch.ones_like(z), "relu": torch.heaviside(z, torch.zeros_like(z)),
                 "gelu": normal_below + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi),
                 "silu": sigmoid + z * sigmoid * (1.0 - sigmoid)}[case["act"]]
        gz = t["gradOutput"] * slope
        out["gradInput"] = torch.cat([torch.einsum("ro,oi->ri", gz[p], weight[g]) for g, p in enumerate(part)])
        out["gradWeight"] = torch.stack([torch.einsum("ro,ri->oi", gz[p], x[p]) for p in part]).reshape(t["weight"].shape)
        out["gradBias"] = torch.stack([gz[p].sum(0) for p in part]).reshape(t["bias"].shape)
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    way = case["way"]
    forward, backward = way != "backward", way != "forward"
    if case["op"] == "norm":
        n, d, r = case["rows"] * case["size"], case["size"], case["rows"]
        # x, weight; the bias and y, or gradOutput and the three gradients; the statistics where they come from another call
        values = n + d + forward * (d + n) + backward * (2 * n + 2 * d) + (way == "backward") * 2 * r
        return {"bytes": 4 * values, "flops": n * (8 * forward + 12 * backward)}
    i, o = case["inputs"], case["outputs"]
    if case["op"] == "linear":
        r, live, groups, residual = case["rows"], 1, 1, case["residual"] and forward
    else:
        counts = counts_of(case)
        r, live, groups, residual = case["tokens"], int((counts > 0).sum()), case["groups"], False
    # x; the weights of groups that have rows; the bias, the residual and y; gradOutput and the three gradients; what a call has kept
    values = r * i + live * i * o + forward * (live * o + r * o * (1 + residual)) + backward * (r * o + r * i + groups * (i + 1) * o) + \
        (way == "backward") * r * o
    if way == "backward" and case["act"] == "none":
        values -= r * o
    return {"bytes": 4 * values, "flops": 2 * r * i * o * (forward + 2 * backward)}
