"""The label head over a large label set (ops.vocab_*): against the formulas in 64 bits with bounds on every element, and what a
program does around it.

Bounds.  A logit is a sum of d products of fp32 accumulation (each addition off by at most 2^-24 of the sum of magnitudes, which is at
most |x_i| |W_v|), fp32 inputs besides as two fp16 pieces (three parts of 2^-22 or less of a product: 2^-20), and is kept in units of
log 2 (two roundings): delta_i.  A probability is off by 2 delta_i of itself, D besides by half a step of fp16 (2^-11; two pieces:
2^-21) or 2^-25 of 2^-14 of the largest |g|; a gradient is a sum of N such terms in steps of 32: (N / 32 + 40) 2^-24 of
the sum of magnitudes, and half a step of its own type."""
import ctypes as C
import math

import pytest
import torch

from pin_slam_amd import _lib, ops

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
F32 = 2.0 ** -24


# ------------------------------------------------------------------------------------------------ refusals (no GPU needed)
@pytest.mark.parametrize("x, w, b, word", [
    ((4, 8), (5, 7), None, "dim"),
    ((4,), (5, 4), None, "dim"),
    ((4, 8), (0, 8), None, "at least one label"),
    ((4, 0), (5, 0), None, "at least one label"),
    ((4, 8), (5, 8), (4,), "bias"),
    ((4, 8), (5, 8), (5,), "device"),
])
def test_shapes_are_refused(x, w, b, word):
    with pytest.raises(RuntimeError, match=word):
        ops.vocab_predict(torch.zeros(x), torch.zeros(w), None if b is None else torch.zeros(b))


@pytest.mark.parametrize("xt, wt, bt", [(torch.float64,) * 3, (torch.float32, torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16, torch.float32)])
def test_types_are_refused(xt, wt, bt):
    with pytest.raises(RuntimeError, match="float"):
        ops.vocab_nll(torch.zeros(2, 3, dtype=xt), torch.zeros(4, 3, dtype=wt), torch.zeros(4, dtype=bt), torch.zeros(2, dtype=torch.int32))


def test_entry_points_refuse_bad_arguments():
    """The C entry points' own checks (host code: no GPU is needed to be refused)."""
    L = _lib.lib()
    at = 1 << 20

    def head(**kw):
        h = _lib.VocabHead(at, at, at, 64, 64, 128, 256, 64, 0)
        for k, v in kw.items():
            setattr(h, k, v)
        return C.byref(h)
    need = L.pin_vocab_workspace_bytes(128, 256, 64, 0, 1)
    assert need > 0
    for bad in (dict(n=-1), dict(vocab=0), dict(dim=0), dict(dtype=3), dict(x=None), dict(weight=None), dict(x_stride=63), dict(weight_stride=1),
                dict(n=(1 << 22) + 1), dict(vocab=(1 << 22) + 1), dict(dim=(1 << 16) + 1)):
        assert L.pin_vocab_nll_step(head(**bad), at, at, at, at, at, at, at, at, need, None) < 0, bad
        assert L.pin_vocab_predict(head(**bad), at, at, at, need, None) < 0, bad
    assert L.pin_vocab_nll_step(head(), at, at, at, at, at, at, at, at, need - 256, None) < 0  # workspace too small
    assert L.pin_vocab_nll_step(head(), at, at, at, at, at, at, at, at + 8, need, None) < 0    # not from a multiple of 256 on
    assert L.pin_vocab_nll_step(head(), None, at, at, at, at, at, at, at, need, None) < 0
    assert L.pin_vocab_nll_grad(head(), at, None, at, at, at, at, at, need, None) < 0
    assert L.pin_vocab_nll(head(), at, None, at, at, need, None) < 0
    assert L.pin_vocab_predict(head(), None, at, at, need, None) < 0
    assert L.pin_vocab_workspace_bytes(0, 5, 5, 0, 1) >= 0 and L.pin_vocab_workspace_bytes(1, 1, 1, 0, 1) > 0
    assert L.pin_vocab_workspace_bytes(1, 0, 1, 0, 1) < 0 and L.pin_vocab_workspace_bytes(1, 1, 1, 5, 0) < 0


# ------------------------------------------------------------------------------------------------ on the GPU
def _inputs(n, vocab, dim, dtype, seed, masked=False, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    w = r(vocab, dim) * dim ** -0.5
    b = r(vocab) * 0.3
    labels = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    if masked:
        off = torch.rand(vocab, device="cuda", generator=gen) < 0.2
        off[0] = False
        b = torch.where(off, torch.full_like(b, -math.inf), b)
        labels = torch.where(off[labels], torch.zeros_like(labels), labels)
        labels[torch.rand(n, device="cuda", generator=gen) < 0.3] = -1
    x = r(n, dim) + 4 * w[labels.clamp(min=0)]
    g = r(n) / max(1, n)
    return (x * scale).to(dtype), (w / scale).to(dtype), b.to(dtype), labels.to(torch.int32), g


def _reference(x, w, b, labels, g):
    """Everything in 64 bits, and for each output the sums of magnitudes its bound is made of."""
    x, w = x.double(), w.double()
    s = x @ w.t() + (b.double() if b is not None else 0)
    lse = torch.logsumexp(s, 1)
    has = labels >= 0
    at = labels.clamp(min=0).long()[:, None]
    nll = torch.where(has, lse - s.gather(1, at)[:, 0], torch.zeros_like(lse))
    d = torch.exp(s - lse[:, None])
    d.scatter_add_(1, at, -torch.ones_like(lse)[:, None])
    d = d * torch.where(has & (lse > -math.inf), g.double(), torch.zeros_like(lse))[:, None]
    d = torch.where(has[:, None] & (lse > -math.inf)[:, None], d, torch.zeros_like(d))
    return s, lse, nll, d


def _delta(x, w, s, lse):
    """Bound of a row's logits."""
    big = x.double().norm(dim=1) * w.double().norm(dim=1).max()
    pieces = 2.0 ** -20 if x.dtype == torch.float32 else 0.0
    finite = torch.where(torch.isfinite(s), s.abs(), torch.zeros_like(s)).amax(1)
    return big * (pieces + (x.shape[1] + 8) * F32) + 4 * F32 * (finite + 1)


def _check(x, w, b, labels, g, got):
    s, lse, nll, d = _reference(x, w, b, labels, g)
    delta = _delta(x, w, s, lse)
    stat = delta + 8 * F32 * (lse.abs().nan_to_num(posinf=0, neginf=0) + 1)
    assert ((got[1].double() - lse).abs() <= stat).all(), ((got[1].double() - lse).abs() / stat).max()
    assert ((got[0].double() - nll).abs() <= 2 * stat).all(), ((got[0].double() - nll).abs() / stat).max()
    if len(got) == 2:
        return
    two = x.dtype == torch.float32
    rp = 2.0 ** -20 if two else 2.0 ** -11
    # (D below 2^-14 of its scale, which is at most 2^-14 of the largest |g|, in fp16's subnormals; two pieces: their sum)
    sub = g.abs().double().max() * 2.0 ** (-39 if not two else -50)
    # (the label's entry is g (p - 1): off by 2 delta of p, however near p is to 1)
    err = torch.exp(s - lse[:, None]).nan_to_num() * g.abs()[:, None] * (2 * stat[:, None]) * (d != 0) + d.abs() * rp + sub * (d != 0)
    eps = torch.finfo(x.dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25}.get(x.dtype, 2.0 ** -140)
    for name, out, full, mag, lost, terms, top in (
            ("dx", got[2], d @ w.double(), d.abs() @ w.double().abs(), err @ w.double().abs(), w.shape[0], d.abs().sum(1, keepdim=True) * w.double().abs().max()),
            ("dw", got[3], d.t() @ x.double(), d.t().abs() @ x.double().abs(), err.t() @ x.double().abs(), x.shape[0], d.t().abs().sum(1, keepdim=True) * x.double().abs().max()),
            ("db", got[4], d.sum(0), d.abs().sum(0), err.sum(0), x.shape[0], None)):
        if out is None:
            continue
        tol = lost + mag * (terms / 32 + 40) * F32 + eps * (full.abs() + lost) + tiny
        if top is not None:  # (the transposed operand in fp16 times a power of two of its tensor: 2^-40 of the largest value; two pieces 2^-21 of each)
            tol = tol + top * 2.0 ** -39 + (mag * 2.0 ** -20 if two else 0)
        off = (out.double() - full).abs()
        assert (off <= tol).all(), (name, (off / tol).max().item(), out.shape)


SHAPES = [(1, 1, 1), (1, 33, 16), (3, 5, 7), (2, 1000, 3), (64, 128, 64), (129, 257, 65), (127, 1000, 50), (256, 150, 64), (130, 5000, 200), (1000, 40, 300),
          (513, 1025, 128), (40, 20011, 96), (300, 3000, 520), (2049, 8191, 72), (260, 777, 180), (900, 1500, 256)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("masked", [False, True])
def test_nll_and_gradients(shape, dtype, masked):
    x, w, b, labels, g = _inputs(*shape, dtype, sum(shape), masked)
    _check(x, w, b, labels, g, ops.vocab_nll_step(x, w, b, labels, g))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [40, 260])
def test_several_pieces_of_the_vocabulary(dtype, dim):
    x, w, b, labels, g = _inputs(1500, 70001, dim, dtype, 3, True)
    _check(x, w, b, labels, g, ops.vocab_nll_step(x, w, b, labels, g))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_no_bias_and_strided_rows(dtype):
    """Views into wider tables, at offsets and strides of 16 bytes and of one element; the columns around them hold NaN."""
    x, w, b, labels, g = _inputs(200, 300, 64, dtype, 4)
    for pad, first in ((64, 8), (7, 3), (1, 0)):
        wide = [torch.full((t.shape[0], 64 + pad + first), math.nan, dtype=dtype, device="cuda") for t in (x, w)]
        views = [t[:, first:first + 64] for t in wide]
        for v, t in zip(views, (x, w)):
            v.copy_(t)
        _check(x, w, None, labels, g, ops.vocab_nll_step(views[0], views[1], None, labels, g))
        assert ops.vocab_nll_step(views[0], views[1], None, labels, g)[4] is None
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.vocab_nll(x.t().contiguous().t(), w, b, labels)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.vocab_nll(x[:1].expand(5, 64), w, b, labels[:5])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [130, 400])
def test_the_two_calls_and_repeats(dtype, dim):
    """The step's loss is vocab_nll's bit for bit; the gradient of a given lse keeps the same bounds; every call repeats its bits, whatever
    an earlier one left in the workspace."""
    x, w, b, labels, g = _inputs(700, 3001, dim, dtype, 5, True)
    nll, lse, *grads = ops.vocab_nll_step(x, w, b, labels, g)
    ws = ops.vocab_workspace(700, 3001, dim, dtype)
    first = None
    for _ in range(2):
        ws.fill_(0xFF)
        a, l = ops.vocab_nll(x, w, b, labels, ws=ws)
        assert torch.equal(a, nll) and torch.equal(l, lse)
        ws.fill_(0xFF)
        alone = ops.vocab_nll_grad(x, w, b, labels, l, g, ws=ws)
        _check(x, w, b, labels, g, (a, l, *alone))
        first = first or alone
        ws.fill_(0xFF)
        for p, q in zip((*alone, *ops.vocab_nll_step(x, w, b, labels, g, ws=ws)), (*first, nll, lse, *grads)):
            assert torch.equal(p, q)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e-6, 1e5])
def test_magnitudes(dtype, scale):
    """Inputs far from 1, upstream gradients over twelve powers of ten, one row and one label a thousand times the others."""
    x, w, b, labels, g = _inputs(300, 700, 96, dtype, 6, False, scale)
    w[5] *= 0.001
    x[7] *= 0.001
    g = g * 10.0 ** torch.linspace(-12, 0, 300, device="cuda")
    s, lse, nll, d = _reference(x, w, b, labels, g)
    got = ops.vocab_nll_step(x, w, b, labels, g)
    stat = _delta(x, w, s, lse) + 8 * F32 * (lse.abs() + 1)
    assert ((got[1].double() - lse).abs() <= stat).all() and ((got[0].double() - nll).abs() <= 2 * stat).all()
    for out, full in zip(got[2:], (d @ w.double(), d.t() @ x.double(), d.sum(0))):
        assert (out.double() - full).norm() <= (2e-6 if dtype == torch.float32 else 2.0 ** -8) * full.norm()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [40, 64, 320])
def test_rows_without_a_label_take_no_part(dtype, dim):
    """NaN and infinities in rows without a label reach no gradient; without any label all gradients are zero."""
    x, w, b, labels, g = _inputs(300, 500, dim, dtype, 7)
    none = torch.zeros(300, dtype=torch.bool, device="cuda")
    none[::3] = True
    labels[none] = -1
    clean = ops.vocab_nll_step(x, w, b, labels, g)
    x[none] = torch.tensor([math.nan, math.inf, -math.inf], device="cuda").to(dtype).repeat(100)[:int(none.sum())][:, None]
    g[none] = math.nan
    got = ops.vocab_nll_step(x, w, b, labels, g)
    assert (got[0][none] == 0).all() and (got[2][none] == 0).all()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2]) and torch.equal(got[4], clean[4])
    assert torch.equal(got[3], clean[3])
    plain = ops.vocab_nll(x, w, b, labels)
    assert torch.equal(plain[0], clean[0]) and torch.equal(plain[1].nan_to_num(posinf=0, neginf=0)[~none], clean[1][~none])
    for t in ops.vocab_nll_step(x, w, b, torch.full_like(labels, -7), g)[2:]:
        assert (t == 0).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [40, 64, 320])
def test_a_labelled_row_that_is_not_finite_is_seen(dtype, dim):
    x, w, b, labels, g = _inputs(200, 300, dim, dtype, 8)
    x[10, 3] = math.nan
    nll, lse, dx, dw, db = ops.vocab_nll_step(x, w, b, labels, g)
    assert nll.isnan().nonzero().flatten().tolist() == [10] and dx[10].isnan().all() and not dx[11].isnan().any()
    assert dw.isnan().any() and db.isnan().any()


@gpu
@pytest.mark.parametrize("low", [-math.inf, -3e38])
def test_labels_that_are_switched_off(low):
    x, w, b, labels, g = _inputs(150, 400, 64, torch.float32, 9)
    b[:] = low
    nll, lse, dx, dw, db = ops.vocab_nll_step(x, w, b, labels, g)
    assert (lse == -math.inf).all() and (nll == math.inf).all()
    assert not dx.any() and not dw.any() and not db.any()
    label, logprob = ops.vocab_predict(x, w, b)
    assert (label == -1).all() and (logprob == -math.inf).all()
    b[17] = 0.5  # one is left: certain
    labels[:] = 17
    nll, lse, dx, dw, db = ops.vocab_nll_step(x, w, b, labels, g)
    assert (nll.abs() < 1e-5).all() and dx.abs().max() < 1e-5
    label, logprob = ops.vocab_predict(x, w, b)
    assert (label == 17).all() and (logprob == 0).all()
    labels[3] = 18  # a row whose own label is off: its loss is infinite, its gradient p - 1 as of any other
    nll, lse, dx, dw, db = ops.vocab_nll_step(x, w, b, labels, g)
    assert nll[3] == math.inf and torch.allclose(dx[3], g[3] * (w[17] - w[18]), rtol=1e-5, atol=1e-7)


@gpu
def test_labels_out_of_range_are_flagged():
    x, w, b, labels, g = _inputs(100, 130, 32, torch.float32, 10)
    ops.status(clear=True)
    labels[5] = 130
    labels[6] = 2 ** 31 - 1
    nll, _, dx, dw, db = ops.vocab_nll_step(x, w, b, labels, g)
    assert nll.isnan().nonzero().flatten().tolist() == [5, 6] and not dx[5:7].any() and not dw.isnan().any()
    with pytest.raises(RuntimeError, match="label"):
        ops.raise_on_status(ops.status())
    assert ops.status() == 0
    with pytest.raises(RuntimeError, match="int32"):
        ops.vocab_nll(x, w, b, labels.long())
    with pytest.raises(RuntimeError, match="labels"):
        ops.vocab_nll(x, w, b, labels[:50])
    with pytest.raises(RuntimeError, match="workspace"):
        ops.vocab_nll(x, w, b, labels, ws=torch.empty(16, dtype=torch.uint8, device="cuda"))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(dtype):
    x, w, b, labels, g = _inputs(4, 70, 33, dtype, 11)
    nll, lse, dx, dw, db = ops.vocab_nll_step(x[:0], w, b, labels[:0], g[:0])
    assert nll.shape == lse.shape == (0,) and dx.shape == (0, 33) and not dw.any() and not db.any()
    assert ops.vocab_predict(x[:0], w, b)[0].shape == (0,) and ops.vocab_nll(x[:0], w, b, labels[:0])[0].shape == (0,)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 131, 64), (1, 70001, 512), (2, 33, 5), (5, 20011, 300), (16, 4096, 256), (17, 4097, 260), (64, 3001, 768), (33, 515, 1030), (20, 131072, 40), (3, 65600, 24), (65, 700, 515),
                                   (300, 1203, 64), (5000, 150, 50)])
@pytest.mark.parametrize("masked", [False, True])
def test_predict(shape, dtype, masked):
    """The label has the largest logit within the bound of the logits, its log-probability follows, and the lowest of equal ones wins."""
    x, w, b, _, _ = _inputs(*shape, dtype, 20 + sum(shape), masked)
    if shape[1] > 40:  # equal rows: equal logits, whatever the arithmetic
        w[shape[1] // 2:shape[1] // 2 + 9] = w[3]
        b[shape[1] // 2:shape[1] // 2 + 9] = b[3]
        x[0] = 6 * w[3]
        b[3:4] = b[shape[1] // 2:shape[1] // 2 + 9] = 8.0
    label, logprob = ops.vocab_predict(x, w, b)
    s = x.double() @ w.double().t() + b.double()
    lse = torch.logsumexp(s, 1)
    delta = _delta(x, w, s, lse)
    best, at = s.max(1)
    mine = s.gather(1, label.long()[:, None])[:, 0]
    assert (best - mine <= 2 * delta).all()
    assert ((logprob.double() - (best - lse)).abs() <= 3 * delta + 8 * F32 * (lse.abs() + 1)).all()
    clear = s.topk(min(2, shape[1]), 1).values
    sure = clear[:, 0] - clear[:, -1] > 2 * delta
    assert torch.equal(label[sure].long(), at[sure])
    if shape[1] > 40:
        assert label[0] == 3


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 131, 64), (7, 20001, 300), (16, 70001, 33), (31, 131073, 72), (33, 66000, 130), (64, 1000, 515), (65, 1000, 515)])
def test_nll_of_a_few_rows(shape, dtype):
    x, w, b, labels, g = _inputs(*shape, dtype, 40 + sum(shape), True)
    _check(x, w, b, labels, g, ops.vocab_nll(x, w, b, labels))
    wide = torch.full((shape[1], shape[2] + 1), math.nan, dtype=dtype, device="cuda")
    wide[:, 1:] = w
    _check(x, w, None, labels, g, ops.vocab_nll(x, wide[:, 1:], None, labels))


@gpu
def test_predict_rows_that_are_not_finite():
    x, w, b, _, _ = _inputs(40, 300, 64, torch.float32, 12)
    x[3, 0] = math.nan
    x[4] = math.inf
    label, logprob = ops.vocab_predict(x, w)
    assert label[3] == -1 and label[4] == -1 and logprob[3:5].isnan().all()
    assert (label[5:] >= 0).all() and torch.isfinite(logprob[5:]).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_captured_calls_that_share_a_workspace(dtype):
    """Two captured steps on one workspace, replayed in turn with eager work between: every replay equals the eager result."""
    sets = [_inputs(n, v, 72, dtype, n, True) for n, v in ((200, 900), (333, 2000))]
    ws = ops.vocab_workspace(333, 2000, 72, dtype)
    graphs, outs = [], []
    for x, w, b, labels, g in sets:
        ops.vocab_nll_step(x, w, b, labels, g, ws=ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((*ops.vocab_nll_step(x, w, b, labels, g, ws=ws), *ops.vocab_predict(x, w, b, ws=ws)))
        graphs.append(graph)
    for k in range(3):
        for x, w, b, labels, g in sets:
            x.mul_(0.9)
            g.mul_(-1.5)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (x, w, b, labels, g), out in zip(sets, outs):
            for p, q in zip(out, (*ops.vocab_nll_step(x, w, b, labels, g), *ops.vocab_predict(x, w, b))):
                assert torch.equal(p, q), k
        torch.cuda.synchronize()


@gpu
def test_another_stream():
    x, w, b, labels, g = _inputs(400, 2000, 100, torch.bfloat16, 14)
    want = ops.vocab_nll_step(x, w, b, labels, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.vocab_nll_step(x, w, b, labels, g)
    side.synchronize()
    for p, q in zip(want, got):
        assert torch.equal(p, q)


@gpu
def test_gradient_against_differences():
    """d nll / d x_ik by central differences of the head itself in fp32: a step of 2^-5 leaves an error of the third derivative (at most
    |W|^3 h^2 / 6 with |W_v| <= 1.5 here) and twice the logits' bound over the step."""
    x, w, b, labels, _ = _inputs(6, 90, 12, torch.float32, 15)
    w = w * (1.0 / w.norm(dim=1).max())
    ones = torch.ones(6, device="cuda")
    _, lse, dx, dw, db = ops.vocab_nll_step(x, w, b, labels, ones)
    h = 2.0 ** -5
    s = x.double() @ w.double().t() + b.double()
    noise = 4 * (_delta(x, w, s, lse.double()).max().item() + 8 * F32 * (s.abs().max().item() + 1)) / (2 * h) + h * h / 6 * 1.0
    for k in range(12):
        e = torch.zeros_like(x)
        e[:, k] = h
        up, down = (ops.vocab_nll(x + q * e, w, b, labels)[0].double() for q in (1, -1))
        assert ((up - down) / (2 * h) - dx[:, k].double()).abs().max() < noise, k


@gpu
def test_training_a_head_runs_as_its_user_would():
    """Features -> NLL with gradients -> AdamW with 8-bit moments on weight and bias, captured into one graph and replayed, the labels then
    predicted: the pieces fit together (buffers, streams, types), the replays equal the eager run bit for bit."""
    def make():
        torch.manual_seed(0)
        w = (torch.randn(1203, 64, device="cuda") * 0.1).bfloat16()
        b = torch.zeros(1203, dtype=torch.bfloat16, device="cuda")
        x = torch.randn(512, 64, device="cuda").bfloat16()
        labels = torch.randint(-1, 1203, (512,), device="cuda").to(torch.int32)
        return x, w, b, labels, ops.AdamW([w, b], lr=0.01, weight_decay=[0.01, 0.0], state_bits=8, seed=1), torch.full((512,), 1 / 512, device="cuda")

    def step(x, w, b, labels, opt, g):
        nll, _, dx, dw, db = ops.vocab_nll_step(x, w, b, labels, g)
        opt.step([dw, db])
        return nll, dx
    eager, cap = make(), make()
    for s in (eager, cap):
        step(*s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*cap)
    for _ in range(3):
        graph.replay()
        want = step(*eager)
        torch.cuda.synchronize()
        for p, q in zip((*out, cap[1], cap[2]), (*want, eager[1], eager[2])):
            assert torch.equal(p, q)
    assert eager[4].steps == cap[4].steps == 5 - 1
    label, logprob = ops.vocab_predict(cap[0], cap[1], cap[2])
    assert ((label >= 0) & (label < 1203)).all() and (logprob <= 0).all()


@gpu
@pytest.mark.parametrize("shape", [(3, 13203, 16), (70, 5001, 64), (130, 900, 200), (5, 4100, 250), (67, 3001, 257), (200, 999, 520)])
def test_float16_dx_is_rounded_once_at_the_label(shape):
    """dx_i = g (sum_v p_v W_v - W_label): the label's factor p - 1 is kept in more than fp16, so that what is left is the rounding of the
    result (2^-11), of the other labels' factors (2^-11 of each one's part) and the probabilities' own error: a logit of d products
    and a bias in fp32 (2^-24 (d + 3) of the sum of their magnitudes, twice: of the maximum's too), and some steps of the exponential and the factors (2^-19)."""
    n, vocab, dim = shape
    x, w, b, labels, _ = _inputs(n, vocab, dim, torch.float16, 5, scale=1.0)
    labels = torch.arange(n, device=x.device, dtype=torch.int32) * 7 % vocab
    x = (x.float() + 3.0 * w[labels.long()].float()).to(torch.float16)
    g = torch.rand(n, device=x.device) + 0.5
    dx = ops.vocab_nll_step(x, w, b, labels, g)[2].double()
    X, W, B = x.double(), w.double(), b.double()
    s = X @ W.t() + B
    p = torch.softmax(s, 1)
    hot = torch.zeros_like(p)
    hot[torch.arange(n, device=x.device), labels.long()] = 1.0
    G = g.double()[:, None]
    want = ((p - hot) @ W) * G
    rel = (X.abs() @ W.t().abs() + B.abs()).amax(1, keepdim=True) * (2.0 ** -24 * (dim + 3) * 2) + 2.0 ** -19
    bound = want.abs() * 2.0 ** -11 + 2.0 ** -25 + ((p * (1 - hot)) @ W.abs()) * (G * (2.0 ** -11 + rel)) + ((p * hot) @ W.abs()) * G * rel
    bound = bound + ((p - hot).abs() @ W.abs()) * G * (F32 * (vocab / 32 + 40)) + W.abs().sum(0) * G.max() * 2.0 ** -39  # sums; tiny factors
    assert ((dx - want).abs() <= bound).all(), float(((dx - want).abs() / bound).max())


@gpu
def test_rows_far_apart():
    """Rows 2^23 + 2^17 elements apart: 256 of them pass 32 bits of bytes."""
    n, vocab, dim, ld = 70, 300, 512, (1 << 23) + (1 << 17)
    x, w, b, labels, g = _inputs(n, vocab, dim, torch.bfloat16, 9)
    far = torch.empty(vocab * ld, dtype=torch.bfloat16, device="cuda").view(vocab, ld)[:, :dim]
    far.copy_(w)
    for a, c in zip(ops.vocab_predict(x, w, b) + ops.vocab_nll_step(x, w, b, labels, g), ops.vocab_predict(x, far, b) + ops.vocab_nll_step(x, far, b, labels, g)):
        assert torch.equal(a, c)
    x = torch.cat([x, x, x, x, x])[:vocab]
    far.copy_(x)
    for a, c in zip(ops.vocab_predict(x, w, b), ops.vocab_predict(far, w, b)):
        assert torch.equal(a, c)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2000, 90, 300), (4686, 672, 352)])
def test_few_labels_and_many_rows(shape, dtype):
    x, w, b, labels, g = _inputs(*shape, dtype, 12, masked=True)
    _check(x, w, b, labels, g, ops.vocab_nll_step(x, w, b, labels, g))


@gpu
def test_a_workspace_in_pieces_is_refused():
    x, w, b, labels, g = _inputs(4, 50, 16, torch.float32, 1)
    ws = ops.vocab_workspace(4, 50, 16)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.vocab_predict(x, w, b, ws=torch.empty(2 * ws.numel(), dtype=torch.uint8, device="cuda")[::2])
    with pytest.raises(RuntimeError, match="must hold"):
        ops.vocab_nll_step(x, w, b, labels, g, ws=ws[:100])


@gpu
def test_float32_passes_agree_to_the_last_bit_of_a_logit():
    """Rows that are nearly certain: db at a label is p - 1 of its row (and little of the others), a difference that a step of the label's
    logit (2^-20 at 16) would move by 1e-6 whatever is left of it.  With logits of the same bits in every pass p is 1 / total rounded
    (half a step, 2^-24), and nll = log total (within 2^-21 of itself: logarithm, product) tells the same total: db = expm1(-nll) + the
    other rows' p, whose errors are delta of their size; D is two pieces (2^-21) and summed in fp32."""
    n, vocab, dim = 64, 128, 64
    x, w, b, _, _ = _inputs(n, vocab, dim, torch.float32, 3)
    labels = torch.arange(n, device="cuda", dtype=torch.int32)
    w = torch.nn.functional.normalize(w, dim=1)
    x = w[:n] * 16 + 0.1 * x
    nll, _, _, _, db = ops.vocab_nll_step(x, w, b, labels, torch.ones(n, device="cuda"))
    X, W = x.double(), w.double()
    p = torch.softmax(X @ W.t() + b.double(), 1)
    others = p.sum(0)[:n] - p.diagonal()
    label = torch.expm1(-nll.double())
    delta = 2 * (X.norm(dim=1).max() * W.norm(dim=1).max() + b.double().abs().max()) * (dim * F32 + 2.0 ** -19)
    bound = 2 * F32 + label.abs() * (2.0 ** -20 + 42 * F32) + others * (2 * delta + 2.0 ** -20 + 42 * F32) + n * 2.0 ** -39
    off = (db.double()[:n] - (label + others)).abs()
    assert (off <= bound).all(), float((off / bound).max())
