"""Performance cases of what a routed feed-forward layer needs around its products, and of the optimiser that trains it: `nn.Router`, `nn.Dispatch`,
`nn.Combine` and `optim.AdamW`.

    listed()            the cases timed by name
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what the program holds before the call
    run(state)          one pass and its outputs: by the framework's modules where `own` is true, else in plain torch operations
    exact(case, seed)   the outputs from the definitions in 64 bits
    work(case)          bytes and floating-point operations the pass cannot do without

Four operators (`case["op"]`):

    router    the `k` largest of `experts` scores of each token, and softmax weights over them (`normalize`) or over all scores.  Scores of minus
              infinity belong to closed experts (`closed`: their share); the last `padded` tokens have none open.  Expert numbers start at 1, 0: none
    dispatch  rows of `size` values copied to the experts they go to: sorted by expert, then token.  `dropped` slots and the last `padded` tokens go
              to none.  With the rows come how many each expert has, on the host, and the place of each slot's row (from 1, 0: none)
    combine   each token's rows from its experts, times their weights, summed, plus a `residual` where the case has one
    adamw     a step of Adam with decoupled weight decay over many tensors, the moments in 32 or in 8 `bits`

`way`: "forward", "backward" (from what a forward pass has left) or "step" (both).  Values are FP32, as all of the framework's tensors are, numbers of
experts and places among them.

Moments in 8 bits: blocks of 256 values of a tensor have a scale each for the mean and for the square root of the mean square.  A code c stands for
(f(b + c 2^s) - f(b)) scale, f(i) the FP32 value of the bits i and b those of 2^-16, with s = 20 for the mean, whose codes are a sign and 7 bits, and s = 19 for
the square root, whose codes are 8 bits.  Codes are rounded up or down at random in proportion to the distance, by 16 bits each of a hash of the value's place,
the tensor's number, the step's number and a seed."""
import math

import numpy as np
import torch

own = False

RATE, BETA1, BETA2, EPSILON, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01

# the weights and biases of the repository's AlexNet-style classifier
ALEXNET = [(64, 3 * 11 * 11), (64,), (192, 64 * 5 * 5), (192,), (384, 192 * 3 * 3), (384,), (256, 384 * 3 * 3), (256,), (256, 256 * 3 * 3), (256,),
           (4096, 9216), (4096,), (4096, 4096), (4096,), (1000, 4096), (1000,)]
# a routed block: a norm, a router and eight experts of two products
EXPERTS = [(2048,), (2048,), (8, 2048), (8,), (8, 1408, 2048), (8, 1408), (8, 2048, 1408), (8, 2048)]


def listed():
    return [
        # one token while answering: latency alone
        {"name": "router_forward_token", "op": "router", "way": "forward", "tokens": 1, "experts": 64, "k": 8, "normalize": True, "closed": 0.0, "padded": 0},
        # a long prompt or a batch of them, many experts
        {"name": "router_forward_prompt", "op": "router", "way": "forward", "tokens": 32768, "experts": 256, "k": 8, "normalize": True, "closed": 0.0,
         "padded": 0},
        # a training step over a padded batch, some experts closed, weights of the whole softmax
        {"name": "router_step_ragged", "op": "router", "way": "step", "tokens": 7001, "experts": 77, "k": 6, "normalize": False, "closed": 0.1, "padded": 333},
        # a few sequences while answering: latency, the host's wait for the counts included
        {"name": "dispatch_forward_few", "op": "dispatch", "way": "forward", "tokens": 24, "size": 4096, "k": 8, "experts": 64, "padded": 0, "dropped": 0},
        # a training step, two experts a token: bandwidth
        {"name": "dispatch_step_wide", "op": "dispatch", "way": "step", "tokens": 8192, "size": 4096, "k": 2, "experts": 16, "padded": 0, "dropped": 0},
        # rows that no 16-byte access divides, a padded batch, slots dropped by a capacity
        {"name": "dispatch_step_ragged", "op": "dispatch", "way": "step", "tokens": 1537, "size": 333, "k": 4, "experts": 37, "padded": 100, "dropped": 211},
        # a few sequences while answering, back into the residual stream
        {"name": "combine_forward_few", "op": "combine", "way": "forward", "tokens": 24, "size": 4096, "k": 8, "experts": 64, "padded": 0, "dropped": 0,
         "residual": True},
        # training, eight experts a token: bandwidth
        {"name": "combine_backward_large", "op": "combine", "way": "backward", "tokens": 8192, "size": 2048, "k": 8, "experts": 64, "padded": 0, "dropped": 0,
         "residual": False},
        # odd sizes, tokens and slots without an expert
        {"name": "combine_step_ragged", "op": "combine", "way": "step", "tokens": 1537, "size": 333, "k": 4, "experts": 37, "padded": 100, "dropped": 211,
         "residual": True},
        # the classifier's 61 million parameters in 16 tensors, two of which are most of them: bandwidth
        {"name": "adamw_32_classifier", "op": "adamw", "bits": 32, "net": "alexnet"},
        # a routed block's parameters, moments in 8 bits
        {"name": "adamw_8_experts", "op": "adamw", "bits": 8, "net": "experts"},
        # many small tensors of any length, side by side in one storage
        {"name": "adamw_32_many", "op": "adamw", "bits": 32, "net": "mixed", "tensors": 300, "total": 2000003, "mix": 1},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["router", "dispatch", "combine", "adamw"])
        if op == "adamw":
            tensors = _log(rng, 1, 400)
            return {"op": op, "bits": rng.choice([32, 8]), "net": "mixed", "tensors": tensors, "total": _log(rng, tensors, 1 << 25), "mix": rng.randrange(1000)}
        tokens, experts, way = _log(rng, 1, 32768), _log(rng, 2, 512), rng.choice(["forward", "backward", "step"])
        k, padded = rng.randint(1, min(experts, 8)), rng.choice([0, tokens // 7])
        case = {"op": op, "way": way, "tokens": tokens, "experts": experts, "k": k, "padded": padded}
        if op == "router":
            case.update(normalize=rng.random() < 0.6, closed=rng.choice([0.0, 0.2]))
            return case
        case.update(size=_log(rng, 16, 8192), dropped=rng.choice([0, (tokens - padded) * k // 9]))
        if op == "combine":
            case["residual"] = rng.random() < 0.4
        if work(case)["bytes"] <= most:
            return case


def lengths_of(case):
    """Values of each tensor of an "adamw" case."""
    if case["net"] != "mixed":
        return [math.prod(s) for s in {"alexnet": ALEXNET, "experts": EXPERTS}[case["net"]]]
    # a few large ones, many small ones, none empty
    r = np.random.RandomState(case["mix"])
    n, spare = case["tensors"], case["total"] - case["tensors"]
    share = np.exp(2.5 * r.standard_normal(n))
    cuts = np.floor(np.cumsum(share) / share.sum() * spare).astype(np.int64)
    cuts[-1] = spare
    return (np.diff(np.concatenate([[0], cuts])) + 1).tolist()


# ------------------------------------------------------------------ inputs
class _State:
    def __init__(self, case):
        self.case = case


def _routing(case, g):
    """Expert numbers of each slot, as a router leaves them: no expert twice for a token, some experts preferred."""
    tokens, experts, k = case["tokens"], case["experts"], case["k"]
    liking = torch.randn(experts, device="cuda", generator=g)
    chosen = (torch.randn((tokens, experts), device="cuda", generator=g) + liking).sort(1, descending=True).indices[:, :k] + 1
    chosen[tokens - case["padded"]:] = 0
    if case["dropped"]:
        lost = torch.randperm((tokens - case["padded"]) * k, device="cuda", generator=g)[:case["dropped"]]
        chosen.view(-1)[lost] = 0
    return chosen.float()


def _places(experts):
    """Places of the slots' rows once these are sorted by expert (from 1, 0: none), the slots in the order of their rows, and how many there are."""
    ids = experts.reshape(-1)
    has = ids > 0
    order = torch.where(has, ids, torch.full_like(ids, math.inf)).sort(stable=True).indices
    rows = int(has.sum())
    places = torch.zeros_like(ids)
    places[order[:rows]] = torch.arange(1, rows + 1, device=ids.device, dtype=ids.dtype)
    return places.view_as(experts), order[:rows], rows


BLOCK, FLOOR, TOP_M, TOP_S = 256, 2.0 ** -16, 0.9375 - 2.0 ** -16, 0.96875 - 2.0 ** -16


def _inputs(case, seed):
    """Everything the pass reads, drawn on the device from the seed."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    t = {}
    if case["op"] == "router":
        shape = (case["tokens"], case["experts"])
        s = 1.5 * normal(*shape) + normal(case["experts"])
        if case["closed"]:
            shut = torch.rand(shape, device="cuda", generator=g) < case["closed"]
            s = torch.where(shut, torch.full_like(s, -math.inf), s)
        s[case["tokens"] - case["padded"]:] = -math.inf
        t["scores"], t["gradWeights"] = s, normal(case["tokens"], case["k"])
        if case["way"] == "backward":      # what the forward pass has left
            t["weights"], t["experts"] = _weights_of(s, case["k"], case["normalize"])
    elif case["op"] == "adamw":
        lengths = lengths_of(case)
        n = sum(lengths)
        size = torch.repeat_interleave(torch.exp(1.5 * normal(len(lengths)) - 6.0), torch.tensor(lengths, device="cuda"), output_size=n)   # of a tensor's gradients
        t["weight"], t["grad"] = 0.05 * normal(n), size * normal(n)
        mean, root = 0.3 * size * normal(n), size * (0.5 + 0.5 * normal(n).abs())
        t["step"] = torch.tensor([float(100 + seed % 7), 0.0], device="cuda")
        if case["bits"] == 32:
            t["mean"], t["square"] = mean, root * root
        else:
            t["meanCodes"], t["rootCodes"], t["scales"] = _codes_of(case, mean, root)
    else:
        experts = _routing(case, g)
        places, order, rows = _places(experts)
        d = case["size"]
        if case["op"] == "dispatch":
            t["x"], t["experts"] = normal(case["tokens"], d), experts
            t["gradRows"] = normal(rows, d)
            if case["way"] == "backward":
                t["places"] = places
        else:
            t["rows"], t["places"] = normal(rows, d), places
            t["weights"] = torch.softmax(normal(case["tokens"], case["k"]), 1) * (places > 0)
            t["gradOutput"] = normal(case["tokens"], d)
            if case["residual"]:
                t["residual"] = normal(case["tokens"], d)
    return t


def _layout(case):
    """Where the values of all tensors lie among their blocks' places, each value's place in its tensor, and its tensor's number; blocks in all."""
    lengths = np.array(lengths_of(case))
    blocks = -(-lengths // BLOCK)
    first = np.cumsum(blocks) - blocks
    n = torch.from_numpy(lengths).cuda()
    number = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), n, output_size=int(lengths.sum()))
    start = (torch.cumsum(n, 0) - n)[number]
    inside = torch.arange(int(lengths.sum()), device="cuda") - start
    return torch.from_numpy(first).cuda()[number] * BLOCK + inside, inside, number, int(blocks.sum())


def _codes_of(case, mean, root):
    """A state in 8 bits, as some earlier step has left it."""
    at, inside, number, blocks = _layout(case)
    padded = torch.zeros((2, blocks * BLOCK), device="cuda")
    padded[0, at], padded[1, at] = mean, root
    padded = padded.view(2, blocks, BLOCK)
    scales = padded.abs().amax(2) / torch.tensor([[TOP_M], [TOP_S]], device="cuda")
    x = (padded.abs() / scales.clamp(min=1e-30)[:, :, None] + FLOOR).contiguous().view(torch.int32) - 0x37800000
    m = torch.clamp((x[0] + (1 << 19)) >> 20, max=127) + 128 * (padded[0] < 0)
    s = torch.clamp((x[1] + (1 << 18)) >> 19, max=255)
    return m.to(torch.uint8).reshape(-1), s.to(torch.uint8).reshape(-1), scales.t().contiguous()


def prepare(case, seed):
    s = _State(case)
    s.t, s.seed = _inputs(case, seed), seed
    if case["op"] == "adamw" and case["bits"] == 8:
        s.layout = _layout(case)
    if own:
        _modules(s)
    torch.cuda.synchronize()
    return s


def _wrap(gt, t):
    """A torch.GPUTensor over a (contiguous) torch tensor's memory."""
    L = gt.lib()
    words = t.numel() * t.element_size() // 4
    st = L.THGPUStorage_newWithData(t.data_ptr(), words)
    v = gt.GPUTensor(_ptr=L.THGPUTensor_newWithStorage1d(st, 0, words, 1))
    L.THGPUStorage_free(st)
    return v.view(*t.shape) if t.element_size() == 4 else v


def _pieces(flat, lengths):
    """Views of neighbouring stretches of a flat tensor."""
    at = np.cumsum([1] + list(lengths)).tolist()
    return [flat.narrow(1, a, n) for a, n in zip(at, lengths)]


def _modules(s):
    """The case's module or optimiser over the case's tensors, with its results in memory that torch sees too."""
    import mcw_cppamp_torch_b200 as gt
    c, t = s.case, s.t
    if c["op"] == "adamw":
        lengths = lengths_of(c)
        blocks = [-(-n // BLOCK) for n in lengths]
        m = gt.optim.AdamW(_pieces(_wrap(gt, t["weight"]), lengths), _pieces(_wrap(gt, t["grad"]), lengths), learningRate=RATE, beta1=BETA1, beta2=BETA2,
                           epsilon=EPSILON, weightDecay=DECAY, bits=c["bits"], seed=s.seed)
        m.step = _wrap(gt, t["step"])
        if c["bits"] == 32:
            m.mean, m.square = _pieces(_wrap(gt, t["mean"]), lengths), _pieces(_wrap(gt, t["square"]), lengths)
        else:
            m.meanCodes = _pieces(_wrap(gt, t["meanCodes"]), [b * 64 for b in blocks])
            m.rootCodes = _pieces(_wrap(gt, t["rootCodes"]), [b * 64 for b in blocks])
            m.scales = _pieces(_wrap(gt, t["scales"].view(-1)), [b * 2 for b in blocks])
            t["mean"], t["square"] = torch.empty_like(t["weight"]), torch.empty_like(t["weight"])
            s.moments = _pieces(_wrap(gt, t["mean"]), lengths), _pieces(_wrap(gt, t["square"]), lengths)
        s.module = m
        gt.synchronize()
        return
    tokens, k = c["tokens"], c["k"]
    g = {n: _wrap(gt, v) if v.numel() else gt.GPUTensor() for n, v in t.items()}

    def room(name, *shape):
        t[name] = torch.zeros(shape, device="cuda")
        return _wrap(gt, t[name])

    if c["op"] == "router":
        m = gt.nn.Router(k, normalize=c["normalize"])
        m.output = [g[n] if n in g else room(n, tokens, k) for n in ("weights", "experts")]
        m.gradInput = room("gradInput", tokens, c["experts"])
        s.input, s.gradOutput = g["scores"], g["gradWeights"]
    elif c["op"] == "dispatch":
        m = gt.nn.Dispatch(c["experts"])
        m.rows, m.positions = room("rows", tokens * k, c["size"]), g["places"] if "places" in g else room("places", tokens, k)
        m.gradRows = room("gradInput", tokens, c["size"])
        s.input, s.gradOutput = [g["x"], g["experts"]], [g["gradRows"], None]
    else:
        m = gt.nn.Combine()
        m.output = room("output", tokens, c["size"])
        m.gradRows, m.gradWeights = room("gradRows", *t["rows"].shape), room("gradWeights", tokens, k)
        s.input = [g["rows"], g["weights"], g["places"]] + ([g["residual"]] if c["residual"] else [])
        s.gradOutput = g["gradOutput"]
    s.module = m
    gt.synchronize()


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    return {"router": _plain_router, "dispatch": _plain_dispatch, "combine": _plain_combine, "adamw": _plain_adamw}[s.case["op"]](s.case, s.t, s)


def _run_own(s):
    m, c, t = s.module, s.case, s.t
    if c["op"] == "adamw":
        m.update()
        if c["bits"] == 8:
            m.moments(*s.moments)
        return {"weight": t["weight"], "mean": t["mean"], "square": t["square"]}
    got = {}
    if c["way"] != "backward":
        out = m.forward(s.input)
        if c["op"] == "router":
            got = {"weights": t["weights"], "experts": t["experts"]}
        elif c["op"] == "dispatch":
            got = {"rows": t["rows"][:int(out[1].sum())], "counts": out[1], "positions": t["places"]}
        else:
            got = {"output": t["output"]}
    if c["way"] != "forward":
        m.backward(s.input, s.gradOutput)
        got.update({"gradRows": t["gradRows"], "gradWeights": t["gradWeights"]} if c["op"] == "combine" else {"gradInput": t["gradInput"]})
    return got


def _weights_of(x, k, normalize):
    """The weights and numbers of each row's largest scores."""
    top, at = x.sort(dim=1, descending=True, stable=True)
    top, at, has = top[:, :k], at[:, :k], top[:, :k] > -math.inf
    largest = torch.where(has[:, :1], top[:, :1], torch.zeros_like(top[:, :1]))
    e = torch.exp(top - largest)
    total = e.sum(1, keepdim=True) if normalize else torch.exp(x - largest).sum(1, keepdim=True)
    return torch.where(has, e / total, torch.zeros_like(e)), torch.where(has, at + 1, torch.zeros_like(at)).float()


def _plain_router(c, t, s):
    x, out = t["scores"], {}
    if c["way"] == "backward":
        weights, experts = t["weights"], t["experts"]
    else:
        weights, experts = _weights_of(x, c["k"], c["normalize"])
        out = {"weights": weights, "experts": experts}
    if c["way"] != "forward":
        has, at = experts > 0, experts.to(torch.int64)
        g = torch.where(has, t["gradWeights"], torch.zeros_like(weights))
        spread = (g * weights).sum(1, keepdim=True)
        wide = x.new_zeros(x.shape[0], x.shape[1] + 1)             # a column more for the slots without an expert
        if c["normalize"]:
            out["gradInput"] = wide.scatter(1, at, weights * (g - spread))[:, 1:].contiguous()
        else:
            largest = x.amax(1, keepdim=True)
            e = torch.exp(x - torch.where(largest > -math.inf, largest, torch.zeros_like(largest)))
            total = e.sum(1, keepdim=True)
            p = e / torch.where(total > 0, total, torch.ones_like(total))
            out["gradInput"] = p * (wide.scatter(1, at, g)[:, 1:] - spread)
    return out


def _plain_dispatch(c, t, s):
    out = {}
    if c["way"] == "backward":
        places = t["places"]
    else:
        places, order, rows = _places(t["experts"])
        counts = torch.bincount(t["experts"].reshape(-1).to(torch.int64), minlength=c["experts"] + 1)[1:].cpu()
        out = {"rows": t["x"][torch.div(order, c["k"], rounding_mode="floor")], "counts": counts, "positions": places}
    if c["way"] != "forward":
        out["gradInput"] = _rows_of(t["gradRows"], places).sum(1)
    return out


def _rows_of(rows, places):
    """Each slot's row, zeros where it has none: [tokens, k, size]."""
    if not rows.numel():
        return torch.zeros(tuple(places.shape) + (rows.shape[1],), device=rows.device, dtype=rows.dtype)
    at = places.to(torch.int64)
    got = rows[(at - 1).clamp(min=0)]
    return got * (at > 0)[:, :, None]


def _plain_combine(c, t, s):
    w, at, out = t["weights"], t["places"].to(torch.int64), {}
    mine = _rows_of(t["rows"], t["places"])
    if c["way"] != "backward":
        y = (w[:, :, None] * mine).sum(1)
        out["output"] = y + t["residual"] if c["residual"] else y
    if c["way"] != "forward":
        g, has = t["gradOutput"], at.reshape(-1) > 0
        grad = torch.zeros_like(t["rows"])
        grad[at.reshape(-1)[has] - 1] = (w[:, :, None] * g[:, None, :]).reshape(-1, c["size"])[has]
        out["gradRows"], out["gradWeights"] = grad, (mine * g[:, None, :]).sum(2) * (at > 0)
    return out


def _hash(place, number, step, seed):
    """32 bits for each value, as int64."""
    mask = 0xffffffff
    h = (place * 0x9e3779b9 + (((seed & mask) ^ (step * 0x9e3779b9 & mask)) + number * 0x6a09e667)) & mask
    h = ((h ^ (h >> 16)) * 0xb7e15163) & mask
    h = ((h ^ (h >> 15)) * 0xadf85459) & mask
    return h ^ (h >> 16)


def _plain_adamw(c, t, s):
    t["step"][0] += 1
    w, g, steps = t["weight"], t["grad"], t["step"][0].double()
    one, two = 1 - BETA1 ** steps, 1 - BETA2 ** steps
    if c["bits"] == 32:
        t["mean"].mul_(BETA1).add_((1 - BETA1) * g)
        t["square"].mul_(BETA2).add_((1 - BETA2) * (g * g))
        mean, square, root = t["mean"], t["square"], torch.sqrt(t["square"])
        out = {"mean": mean, "square": square}
    else:
        at, inside, number, blocks = s.layout
        scales = t["scales"]

        def value(code, shift, scale):
            bits = (code.to(torch.int32) << shift) + 0x37800000
            return ((bits.view(torch.float32) - FLOOR).view(blocks, BLOCK) * scale[:, None]).view(-1)[at]

        codes = t["meanCodes"].to(torch.int32)
        mean = value(codes & 127, 20, scales[:, 0])
        mean = torch.where((codes & 128).bool()[at], -mean, mean)
        root = value(t["rootCodes"], 19, scales[:, 1])
        mean = BETA1 * mean + (1 - BETA1) * g
        root = torch.sqrt(BETA2 * (root * root) + (1 - BETA2) * (g * g))
        random = _hash(inside, number, steps.long(), s.seed)

        def coded(x, top, shift, noise, most):
            padded = torch.zeros(blocks * BLOCK, device="cuda")
            padded[at] = x
            scale = padded.view(blocks, BLOCK).amax(1) * (1.0 / top)
            scale = torch.where(scale >= 2.0 ** -126, scale, torch.zeros_like(scale))
            inverse = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
            scaled = (padded.view(blocks, BLOCK) * inverse[:, None]).view(-1) + FLOOR
            bits = scaled.view(torch.int32) - 0x37800000
            noisy = torch.zeros_like(bits)
            noisy[at] = ((noise << (shift - 16)) + (1 << (shift - 17))).to(torch.int32)
            return torch.clamp((bits + noisy) >> shift, max=most), scale

        m, scale_m = coded(mean.abs(), TOP_M, 20, random & 0xffff, 127)
        r, scale_s = coded(root, TOP_S, 19, random >> 16, 255)
        negative = torch.zeros_like(m)
        negative[at] = (mean < 0).to(torch.int32)
        t["meanCodes"].copy_(m | (negative << 7))
        t["rootCodes"].copy_(r)
        t["scales"][:, 0], t["scales"][:, 1] = scale_m, scale_s
        kept = value(m, 20, scale_m)
        kept_root = value(r, 19, scale_s)
        out = {"mean": torch.where(negative[at].bool(), -kept, kept), "square": kept_root * kept_root}
    w.mul_(1 - RATE * DECAY).sub_((RATE / one).float() * (mean / (root / torch.sqrt(two).float() + EPSILON)))
    return {"weight": w, **out}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    t = {k: v.double() if v.dtype == torch.float32 else v for k, v in _inputs(case, seed).items()}
    return {"router": _exact_router, "dispatch": _exact_dispatch, "combine": _exact_combine, "adamw": _exact_adamw}[case["op"]](case, t, seed)


def _exact_router(c, t, seed):
    x = t["scores"]
    rest, chosen = x.clone(), []
    for _ in range(c["k"]):                # the largest of what is left, the first of equal ones
        top = rest.max(1, keepdim=True).values
        first = (rest == top).to(torch.int8).argmax(1, keepdim=True)
        chosen.append(torch.where(top == -math.inf, torch.full_like(first, -1), first))
        rest.scatter_(1, first, -math.inf)
    chosen = torch.cat(chosen, 1)
    on = torch.zeros_like(x, dtype=torch.bool)
    for i in range(c["k"]):
        on |= torch.arange(c["experts"], device=x.device) == chosen[:, i:i + 1]
    over = torch.where(on, x, torch.full_like(x, -math.inf)) if c["normalize"] else x
    p = torch.nan_to_num(torch.softmax(over, 1))
    picked = chosen.clamp(min=0)
    weights = p.gather(1, picked) * (chosen >= 0)
    out = {} if c["way"] == "backward" else {"weights": weights, "experts": None}
    if c["way"] != "forward":
        g = torch.zeros_like(x)
        for i in range(c["k"]):
            g += torch.where(torch.arange(c["experts"], device=x.device) == chosen[:, i:i + 1], t["gradWeights"][:, i:i + 1], 0.0)
        out["gradInput"] = p * g - p * torch.einsum("te,te->t", p, g)[:, None]
    return out


def _members(experts, number):
    """Tokens of each expert, in order."""
    return [(experts == e + 1).any(1).nonzero()[:, 0] for e in range(number)]


def _exact_dispatch(c, t, seed):
    members = torch.cat(_members(t["experts"], c["experts"]))
    out = {} if c["way"] == "backward" else {"rows": t["x"].index_select(0, members), "counts": None, "positions": None}
    if c["way"] != "forward":
        out["gradInput"] = torch.zeros_like(t["x"]).index_add_(0, members, t["gradRows"])
    return out


def _exact_combine(c, t, seed):
    token, slot = (t["places"] > 0).nonzero(as_tuple=True)
    at = t["places"][token, slot].long() - 1
    w = t["weights"][token, slot]
    out = {}
    if c["way"] != "backward":
        y = torch.zeros_like(t["gradOutput"]).index_add_(0, token, t["rows"].index_select(0, at) * w[:, None])
        out["output"] = y + t["residual"] if c["residual"] else y
    if c["way"] != "forward":
        g = t["gradOutput"].index_select(0, token)
        out["gradRows"] = torch.zeros_like(t["rows"]).index_copy_(0, at, torch.einsum("rd,r->rd", g, w))
        out["gradWeights"] = torch.zeros_like(t["weights"]).index_put_((token, slot), torch.einsum("rd,rd->r", g, t["rows"].index_select(0, at)))
    return out


def _exact_adamw(c, t, seed):
    steps, g = int(t["step"][0]) + 1, t["grad"]
    if c["bits"] == 32:
        mean, square = torch.lerp(t["mean"], g, 1 - BETA1), torch.lerp(t["square"], g * g, 1 - BETA2)
        out = {"mean": mean, "square": square}
    else:
        at = _layout(c)[0]
        block = at // BLOCK
        low = math.log2(FLOOR)

        def value(code, parts):            # a code's place among the `parts` of each power of two
            code = code.double()
            power = torch.floor(code / parts)
            return torch.ldexp(1.0 + code / parts - power, power + low) - FLOOR

        was_m, was_s = t["meanCodes"][at], t["rootCodes"][at]
        m = value(was_m & 127, 8) * t["scales"][block, 0] * (1.0 - 2.0 * (was_m >> 7).double())
        r = value(was_s, 16) * t["scales"][block, 1]
        mean, square = torch.lerp(m, g, 1 - BETA1), torch.lerp(r ** 2, g ** 2, 1 - BETA2)
        # Which of two neighbouring codes a value gets is a matter of the last bit of the FP32 sum that is rounded: 64 bits do not tell.
        out = {"mean": None, "square": None}
    corrected = torch.sqrt(square / (1 - BETA2 ** steps)) + EPSILON
    return {"weight": t["weight"] * (1 - RATE * DECAY) - RATE * (mean / (1 - BETA1 ** steps)) / corrected, **out}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    forward, backward = case.get("way") != "backward", case.get("way") != "forward"
    if case["op"] == "adamw":
        lengths = lengths_of(case)
        n, blocks = sum(lengths), sum(-(-k // BLOCK) for k in lengths)
        # weights, gradients and the weights again; the moments both ways, or their codes and scales and the values these stand for
        return {"bytes": 12 * n + (16 * n if case["bits"] == 32 else 4 * BLOCK * blocks + 16 * blocks + 8 * n), "flops": (14 if case["bits"] == 32 else 40) * n}
    tokens, k, experts = case["tokens"], case["k"], case["experts"]
    slots, live = tokens * k, tokens - case["padded"]
    if case["op"] == "router":
        # the scores, unless the weights say all that their gradient needs; weights and numbers; gradients of the weights and of the scores
        values = tokens * experts * (forward or not case["normalize"]) + 2 * slots + backward * (slots + tokens * experts)
        return {"bytes": 4 * values, "flops": tokens * experts * (forward + backward) + 4 * slots}
    d, rows = case["size"], live * k - case["dropped"]
    reached = min(live, rows)
    if case["op"] == "dispatch":
        # rows in and out, expert numbers and places; the way back
        values = forward * (reached * d + rows * d + slots) + slots + backward * (rows * d + tokens * d)
        return {"bytes": 4 * values, "flops": max(1, backward * rows * d)}
    # rows, weights and places; a residual, sums; gradients of sums and of both operands
    values = rows * d + 2 * slots + forward * tokens * d * (1 + case["residual"]) + backward * (reached * d + rows * d + slots)
    return {"bytes": 4 * values, "flops": rows * d * (2 * forward + 3 * backward)}
