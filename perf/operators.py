"""The operators of the label head over a large label set and of the optimiser that trains it, as a user's program calls them.

  nll      the negative log-likelihood of a linear head over ``vocab`` labels, with its gradients (one training pass)
  predict  the most probable label of every row and its log-probability (answering)
  adamw    one AdamW step over many tensors, moments in 32 or in 8 bits

``run`` computes an operator in its plain form, or (``own``) through the framework's entry points."""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 256   # elements that share a scale of the 8-bit moments; every tensor begins at a multiple of it
BETA1, BETA2, EPS, LR, DECAY = 0.9, 0.99, 1e-15, 0.01, 0.01
# the decoder of the map at 4 hidden layers of 64: weights and biases in state_dict order
DECODER = "704 64 4096 64 4096 64 4096 64 64 1"


def listed():
    return [
        # a decoder's features against a small label set: latency counts
        {"name": "nll small fp32", "op": "nll", "dtype": "float32", "n": 256, "vocab": 150, "dim": 64, "masked": False},
        # the mapper's batch (16384 samples, 64 hidden units) over a label set of a thousand, some labels switched off
        {"name": "nll batch fp32", "op": "nll", "dtype": "float32", "n": 16384, "vocab": 1203, "dim": 64, "masked": True},
        # the same batch over an open label set, in bf16
        {"name": "nll open set bf16", "op": "nll", "dtype": "bfloat16", "n": 16384, "vocab": 32768, "dim": 64, "masked": False},
        # odd sizes everywhere: no row begins at a multiple of 16 bytes
        {"name": "nll ragged fp16", "op": "nll", "dtype": "float16", "n": 5003, "vocab": 21841, "dim": 195, "masked": True},
        # wide image features distilled into labels: the products carry it
        {"name": "nll wide bf16", "op": "nll", "dtype": "bfloat16", "n": 8192, "vocab": 32768, "dim": 1024, "masked": False},
        # one query against the whole label set: the weights are read once, and that is all there is
        {"name": "predict one bf16", "op": "predict", "dtype": "bfloat16", "n": 1, "vocab": 131072, "dim": 512, "masked": False},
        # a few queries, ragged
        {"name": "predict few fp32", "op": "predict", "dtype": "float32", "n": 19, "vocab": 30011, "dim": 300, "masked": True},
        # every point of a scan labelled
        {"name": "predict scan fp16", "op": "predict", "dtype": "float16", "n": 100000, "vocab": 1203, "dim": 64, "masked": False},
        # the decoder alone: ten small tensors, latency counts
        {"name": "adamw decoder fp32", "op": "adamw", "bits": 32, "param": "float32", "grad": "float32", "sizes": DECODER},
        # the feature table of 2.2 million points and the decoder
        {"name": "adamw map fp32", "op": "adamw", "bits": 32, "param": "float32", "grad": "float32", "sizes": "17600008 " + DECODER},
        # a head over an open label set in bf16 beside two feature tables of five million points, moments in 8 bits
        {"name": "adamw head 8-bit bf16", "op": "adamw", "bits": 8, "param": "bfloat16", "grad": "bfloat16",
         "sizes": "33554432 32768 40000008 40000008"},
        # many ragged tensors, moments in 8 bits
        {"name": "adamw many 8-bit fp32", "op": "adamw", "bits": 8, "param": "float32", "grad": "float32",
         "sizes": " ".join(str(1 + (i * i * 7919 + 31 * i) % 60001) for i in range(150))},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["nll", "nll", "predict", "adamw"])
    if op == "adamw":
        count = _log(rng, 1, 200)
        most = 1.0e8 / count
        sizes = [max(1, _log(rng, 1, max(2, min(most, 4.0e7)))) for _ in range(count)]
        param = rng.choice(["float32", "bfloat16", "float16"])
        return {"op": "adamw", "bits": rng.choice([8, 32]), "param": param, "grad": rng.choice([param, "float32"]),
                "sizes": " ".join(map(str, sizes))}
    while True:
        n, vocab, dim = _log(rng, 1, 16384 if op == "nll" else 100000), _log(rng, 33, 131072), _log(rng, 16, 1024)
        if n * vocab * dim <= 2.7e11 and n * vocab <= 5.5e8:
            return {"op": op, "dtype": rng.choice(sorted(DTYPES)), "n": n, "vocab": vocab, "dim": dim, "masked": rng.random() < 0.4}


# ---------------------------------------------------------------------------------------------------- inputs
def _head(case, seed):
    """A head that has learnt something: a row lies along its label's weights, among noise, so that the label's logit stands
    out of the others'; a quarter of a training batch carries no label; ``masked``: one label in eight is switched off."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n, vocab, dim, dtype = case["n"], case["vocab"], case["dim"], DTYPES[case["dtype"]]
    weight = torch.randn(vocab, dim, device="cuda", generator=gen).mul_(dim ** -0.5)
    bias = torch.randn(vocab, device="cuda", generator=gen).mul_(0.3)
    labels = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    if case["masked"]:
        off = torch.rand(vocab, device="cuda", generator=gen) < 0.125
        off[0] = False
        bias = torch.where(off, torch.full_like(bias, -math.inf), bias)
        labels = torch.where(off[labels], torch.zeros_like(labels), labels)
    noise = torch.randn(n, dim, device="cuda", generator=gen)
    pull = (8.0 if case["op"] == "predict" else 4.0) + 8.0 * torch.rand(n, 1, device="cuda", generator=gen)
    x = noise + pull * weight[labels]
    rest = torch.rand(n, device="cuda", generator=gen)
    return {"case": case, "x": x.to(dtype), "weight": weight.to(dtype), "bias": bias.to(dtype), "labels": labels.to(torch.int32), "rest": rest}


def prepare(case, seed):
    if case["op"] == "adamw":
        return _prepare_adamw(case, seed)
    s = _head(case, seed)
    rest = s.pop("rest")
    if case["op"] == "nll":
        # no label on a quarter of the rows; the weights of the others as of a mean over the samples by their distance
        labelled = rest >= 0.25
        labelled[:1] = True
        s["labels"] = torch.where(labelled, s["labels"], torch.full_like(s["labels"], -1))
        s["grad_nll"] = (0.5 + rest) / labelled.sum()
    else:
        del s["labels"]
    return s


def _layout(case):
    sizes = [int(v) for v in case["sizes"].split()]
    starts, at = [], 0
    for v in sizes:
        starts.append(at)
        at += -(-v // BLOCK) * BLOCK
    return sizes, starts, at


def _prepare_adamw(case, seed):
    """Parameters and gradients, each the views of one buffer in which every tensor begins at a multiple of BLOCK, and
    moments as a few hundred steps leave them: over the tensor's rows their size spreads over some powers of ten."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    sizes, starts, total = _layout(case)
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    for v, a in zip(sizes, starts):
        inside[a:a + v] = True

    def normal():
        return torch.randn(total, device="cuda", generator=gen).mul_(inside)
    spread = torch.randn(-(-total // 64), device="cuda", generator=gen).mul_(1.5).exp_().repeat_interleave(64)[:total].mul_(1e-3)
    param = normal().mul_(0.1).to(DTYPES[case["param"]])
    grad = normal().mul_(spread).to(DTYPES[case["grad"]])
    exp_avg = normal().mul_(spread).mul_(0.3)
    exp_avg_sq = normal().square_().mul_(0.2).add_(0.9).mul_(inside).mul_(spread.square_())
    del spread
    s = {"case": case, "step": 300, "seed": 12345 + seed % 1000, "param": param, "grad": grad, "total": total, "inside": inside}
    if case["bits"] == 32:
        s["exp_avg"], s["exp_avg_sq"] = exp_avg, exp_avg_sq
    else:
        s["exp_avg"], s["exp_avg_scale"] = _squeeze(exp_avg, 8, 0x600000, 0.5)
        s["exp_avg"] = s["exp_avg"].to(torch.float8_e4m3fn)
        s["exp_avg_sq"], s["exp_avg_sq_scale"] = _squeeze(exp_avg_sq, 15, 0x600000, 0.5)
        s["exp_avg_sq"] = s["exp_avg_sq"].to(torch.float8_e5m2)
    if own:
        from pin_slam_amd import ops
        params = [param[a:a + v] for v, a in zip(sizes, starts)]
        grads = [grad[a:a + v] for v, a in zip(sizes, starts)]
        s["optimizer"] = ops.AdamW(params, grads, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case["bits"], seed=s["seed"])
        s["optimizer"].load_state_dict({"step": s["step"], **{k: s[k] for k in s if k.startswith("exp_avg")}})
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _nll(x, weight, bias, labels, grad_nll, dtype):
    x, weight, bias = x.to(dtype), weight.to(dtype), bias.to(dtype)
    logits = x @ weight.t() + bias
    top = logits.amax(1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(1, keepdim=True)
    lse = top + torch.log(total)
    has = (labels >= 0).unsqueeze(1)
    label = labels.clamp(min=0).long().unsqueeze(1)
    nll = torch.where(has, lse - logits.gather(1, label), torch.zeros_like(lse))
    del logits
    p.div_(total)
    p.scatter_add_(1, label, torch.full_like(lse, -1.0))
    p.mul_(torch.where(has, grad_nll.to(dtype).unsqueeze(1), torch.zeros_like(lse)))
    return nll.squeeze(1), lse.squeeze(1), p @ weight, p.t() @ x, p.sum(0)


def _predict(x, weight, bias, dtype):
    logits = x.to(dtype) @ weight.to(dtype).t() + bias.to(dtype)
    top = logits.amax(1, keepdim=True)
    places = torch.arange(logits.shape[1], device=logits.device, dtype=torch.int32)
    label = torch.where(logits == top, places, torch.full_like(places, logits.shape[1])).amin(1)  # ties: the lowest
    return label, -torch.log(torch.exp(logits - top).sum(1))


def _mixed(h):
    """A 32-bit hash of 32-bit numbers held in 64 bits."""
    h = h ^ (h >> 16)
    h = (h * 0x9E3779B1) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0xB7E15163) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _power(exponent):
    """2 ** exponent of normal numbers, exactly, as float32."""
    return ((exponent + 127) << 23).view(torch.float32)


def _exponent(v):
    """floor(log2 v) of normal numbers; -127 for smaller ones."""
    return (v.view(torch.int32) >> 23) - 127


def _squeeze(value, top, fraction, dither):
    """(value / scale, rounded by the dither to 8-bit floating point, as float32; scale a block of 256).  The format's largest
    number is (1 + fraction / 2^23) 2^top with two or three bits of fraction; the scale is the smallest power of two, 2^-100 or
    more, with the block's largest magnitude inside the format."""
    bits = 3 if top == 8 else 2
    low = -6 if top == 8 else -14
    size = value.abs().view(-1, BLOCK)
    largest = size.amax(1)
    e = _exponent(largest) - top
    e = torch.where((largest.view(torch.int32) & 0x7FFFFF) > fraction, e + 1, e).clamp(min=-100)
    scale = _power(e)
    size = (size * _power(-e).unsqueeze(1)).view(-1)
    e = _exponent(size).clamp(min=low) - bits
    n = torch.floor(size * _power(-e) + dither)
    size = n * _power(e)
    if top != 8:  # a second moment that is not zero stays so
        size = torch.where((n == 0) & (value > 0), torch.full_like(size, 2.0 ** (low - bits)), size)
    return torch.where(value < 0, -size, size).clamp(-(1 + fraction / 2 ** 23) * 2.0 ** top, (1 + fraction / 2 ** 23) * 2.0 ** top), scale


def _adamw(s):
    """In place, as an optimiser works.  The order of the operations on the moments is the operator's own: what the 8-bit
    codes round to depends on it at their borders."""
    s["step"] += 1
    t = s["step"]
    g = s["grad"].float()
    m, v = s["exp_avg"].float(), s["exp_avg_sq"].float()
    if s["case"]["bits"] == 8:
        m = (m.view(-1, BLOCK) * s["exp_avg_scale"].unsqueeze(1)).view(-1)
        v = (v.view(-1, BLOCK) * s["exp_avg_sq_scale"].unsqueeze(1)).view(-1)
    one, two = torch.tensor(1.0) - torch.tensor([BETA1, BETA2])
    m = m + (g - m) * one.item()
    v = v * torch.tensor(BETA2).item() + two.item() * g * g
    step = LR / (1.0 - BETA1 ** t) * (m / (torch.sqrt(v) * (1.0 / math.sqrt(1.0 - BETA2 ** t)) + EPS))
    s["param"].copy_(s["param"].float() * (1.0 - LR * DECAY) - step)
    if s["case"]["bits"] == 32:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
        return [s["param"], s["exp_avg"], s["exp_avg_sq"]]
    key = _mixed(_mixed(torch.tensor(s["seed"] & 0xFFFFFFFF, device=g.device)) ^ (t & 0xFFFFFFFF))
    h = _mixed((torch.arange(s["total"], device=g.device) & 0xFFFFFFFF) ^ key)
    for name, value, dither, top in (("exp_avg", m, h & 0xFFFF, 8), ("exp_avg_sq", v, h >> 16, 15)):
        code, scale = _squeeze(value, top, 0x600000, dither.float() * 2.0 ** -16)
        s[name].copy_(code)
        s[name + "_scale"].copy_(scale)
    return [s["param"], s["exp_avg"], s["exp_avg_sq"], s["exp_avg_scale"], s["exp_avg_sq_scale"]]


def run(state):
    case = state["case"]
    if case["op"] == "nll":
        if own:
            from pin_slam_amd import ops
            return ops.vocab_nll_step(state["x"], state["weight"], state["bias"], state["labels"], state["grad_nll"])
        nll, lse, dx, dw, db = _nll(state["x"], state["weight"], state["bias"], state["labels"], state["grad_nll"], torch.float32)
        dtype = state["x"].dtype
        return nll, lse, dx.to(dtype), dw.to(dtype), db.to(dtype)
    if case["op"] == "predict":
        if own:
            from pin_slam_amd import ops
            return ops.vocab_predict(state["x"], state["weight"], state["bias"])
        return _predict(state["x"], state["weight"], state["bias"], torch.float32)
    if own:
        opt = state["optimizer"]
        opt.step()
        if case["bits"] == 32:
            return [state["param"], opt.exp_avg, opt.exp_avg_sq]
        return [state["param"], opt.exp_avg, opt.exp_avg_sq, opt.exp_avg_scale, opt.exp_avg_sq_scale]
    return _adamw(state)


# ---------------------------------------------------------------------------------------------------- work and definition
def work(case):
    if case["op"] == "adamw":
        total = sum(int(v) for v in case["sizes"].split())
        size = {"float32": 4, "bfloat16": 2, "float16": 2}
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": total * (2 * size[case["param"]] + size[case["grad"]] + moments), "flops": 14.0 * total}
    n, vocab, dim = case["n"], case["vocab"], case["dim"]
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "predict":
        return {"bytes": size * (n * dim + vocab * dim + vocab) + 8 * n, "flops": 2.0 * n * vocab * dim}
    return {"bytes": 2 * size * (n * dim + vocab * dim + vocab) + 16 * n, "flops": 6.0 * n * vocab * dim}


def exact(case, seed):
    """From the definitions, in 64 bits: log p = s - lse, d nll_i / d s_iv = p_iv - [v = y_i]."""
    s = prepare(case, seed)
    if case["op"] == "adamw":
        t = s["step"] + 1
        g, p = s["grad"].double(), s["param"].double()
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
        if case["bits"] == 8:
            m = (m.view(-1, BLOCK) * s["exp_avg_scale"].double().view(-1, 1)).flatten()
            v = (v.view(-1, BLOCK) * s["exp_avg_sq_scale"].double().view(-1, 1)).flatten()
        m, v = BETA1 * m + (1 - BETA1) * g, BETA2 * v + (1 - BETA2) * g ** 2
        p = (1 - LR * DECAY) * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
        # (what the 8-bit codes round to hangs on the 32-bit arithmetic at their borders: no value in 64 bits)
        return [p, m, v] if case["bits"] == 32 else [p, None, None, None, None]
    x, w = s["x"].double(), s["weight"].double()
    z = torch.addmm(s["bias"].double(), x, w.t())
    lse = torch.logsumexp(z, 1)
    if case["op"] == "predict":
        best, at = z.max(1)
        return None, best - lse
    rows = torch.nonzero(s["labels"] >= 0).flatten()
    at = s["labels"][rows].long()
    nll = torch.zeros(case["n"], dtype=torch.float64, device="cuda")
    nll[rows] = lse[rows] - z[rows, at]
    d = torch.zeros_like(z)
    d[rows] = torch.exp(z[rows] - lse[rows].unsqueeze(1))
    del z
    d[rows, at] -= 1.0
    d *= s["grad_nll"].double().unsqueeze(1)
    return nll, lse, d @ w, d.t() @ x, d.sum(0)
