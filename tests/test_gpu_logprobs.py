"""The kernels behind zenyx_b200/ops/logprobs.py against 64-bit forms (tests/_logprobs_oracle.py, which derives the
tolerances): types, vocabularies that no vector divides, strides, ties, masks that leave nothing, gradients, graphs, streams."""
import math

import pytest
import torch

import _logprobs_oracle as oracle
from zenyx_b200.ops import _ext, logprobs as ops
from zenyx_b200.ops.logprobs import MAX_VOCAB, distill_topk, distill_topk_fwd_bwd_, token_logprobs

pytestmark = pytest.mark.gpu
NEG = float("-inf")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _status():
    yield
    _ext.check_status()


def _logits(T, V, dtype, seed=0, std=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, V, generator=gen, device="cuda") * std
    return x.to(dtype), torch.randint(0, V, (T,), generator=gen, device="cuda"), gen


def _check_fwd(x, y, K, t=1.0):
    out = token_logprobs(x, y, top_k=K, temperature=t)
    lp, h, top, ids, *_ = oracle.logprobs(x, y, K, t)
    V = x.shape[1]
    if K:
        assert torch.equal(out.top_ids, ids), "alternatives"
        oracle.check(out.top_logprobs, top, oracle.logprob_off(torch.nan_to_num(top, neginf=0.0), h[:, None], V), "top")
    if y is not None:
        oracle.check(out.logprobs, lp, oracle.logprob_off(torch.nan_to_num(lp, neginf=0.0), h, V), "logprobs")
    oracle.check(out.entropy, h, oracle.entropy_off(h, V), "entropy")
    return out


def _check_bwd(x, y, K, t=1.0, parts=("lp", "h", "top"), seed=5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T = x.shape[0]
    a = x.detach().requires_grad_(True)
    out = token_logprobs(a, y, top_k=K, temperature=t)
    grads = {"lp": torch.randn(T, generator=gen, device="cuda"), "h": torch.randn(T, generator=gen, device="cuda")}
    if K:
        grads["top"] = torch.randn(T, K, generator=gen, device="cuda")
    outs = {"lp": out.logprobs, "h": out.entropy, "top": out.top_logprobs}
    use = [p for p in parts if p in grads and outs[p] is not None]
    (got,) = torch.autograd.grad([outs[p] for p in use], a, [grads[p] for p in use])
    ref, off = oracle.logprobs_grad(x, y, K, t, *[grads[p] if p in use else None for p in ("lp", "h", "top")])
    oracle.check(got, ref, off, "gradient")
    return got


SHAPES = [(1, 1), (3, 2), (2, 7), (5, 8), (3, 31), (4, 64), (2, 129), (7, 1000), (3, 4096), (2, 8191), (300, 513),
          (2, 32000), (3, 50257), (1, 128256), (2, 151937), (1, 262147)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", SHAPES)
def test_logprobs_values(dtype, T, V):
    x, y, _ = _logits(T, V, dtype, seed=V)
    if T > 2:
        y[1] = -100
    for K, t in ((0, 1.0), (1, 0.6), (20, 1.0), (128, 2.0)):
        _check_fwd(x, y, min(K, V), t)
    _check_fwd(x, None, min(5, V))
    _check_fwd(x, y.int(), 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", SHAPES)
def test_logprobs_gradient(dtype, T, V):
    x, y, _ = _logits(T, V, dtype, seed=V + 1)
    if T > 2:
        y[1] = -1
    K = min(17, V)
    _check_bwd(x, y, 0, 1.0, ("lp",))
    _check_bwd(x, y, 0, 0.7, ("lp", "h"))
    _check_bwd(x, y, K, 1.3)
    _check_bwd(x, None, K, 1.0, ("h", "top"))
    _check_bwd(x, y, min(128, V), 1.0, ("top",))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5, 640, 8195, 128256])
def test_rows_that_stand_for_nothing(dtype, V):
    x, y, _ = _logits(12, V, dtype, seed=3)
    low = torch.finfo(dtype).min
    x[0] = NEG                                         # nothing is left
    x[1] = NEG
    x[1, V // 2] = 1.5                                 # one token is
    x[2] = low                                         # masked with the type's lowest value: all alike
    x[3] = low
    x[3, 4] = 0.0
    x[4, 2] = float("nan")
    x[5, V - 1] = float("inf")
    x[6] = float("nan")                                # left out: not looked at
    y[6] = -100
    x[7, : V - 3] = NEG                                # fewer tokens than alternatives
    x[8] = torch.finfo(dtype).max
    y[9] = V                                           # out of range: left out
    x[10, ::2] = -0.0
    x[10, 1::2] = 0.0
    x[11] = low
    x[11, 1] = torch.finfo(dtype).max
    K = min(V, 7)
    for t in (1.0, 0.5):
        _check_fwd(x, y, K, t)
    rows = torch.tensor([0, 1, 2, 3, 6, 7, 9, 10, 11], device="cuda")
    y[7] = V - 1
    y[1] = V // 2
    y[3] = 4
    y[11] = 1
    got = _check_bwd(x[rows], y[rows], K)
    assert (got[0] == 0).all() and (got[4] == 0).all() and (got[6] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [512, 9001, 128256])
def test_orders_and_ties(dtype, V):
    """Rows on which a threshold taken from a sample says least: sorted both ways, all alike, blocks alike, all large
    values on one residue of the column, few distinct values."""
    j = torch.arange(V, device="cuda", dtype=torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(1)
    rows = [j / V * 20, -j / V * 20, torch.zeros_like(j), torch.where(j < V // 2, 1.0, 2.0), torch.where(j < V // 2, 2.0, 1.0)]
    for step in (8, 64, 512, 4096):
        rows.append(torch.where(j % step == 3, 5.0 + j / V, -j / V))
    rows.append(torch.randint(0, 3, (V,), generator=gen, device="cuda").float())
    rows.append(torch.where(j % 1024 < 8, 3.0, torch.randn(V, generator=gen, device="cuda")))
    rows.append(torch.where(j >= V - 300, 4.0 + (j % 7), -1.0))
    rows.append(torch.where(j < 300, 4.0 + (j % 7), -1.0))
    x = torch.stack(rows).to(dtype)
    for K in (1, 2, 20, 64, 128):
        _check_fwd(x, None, K)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_addresses(dtype):
    """Rows that start at every address, wider row strides, the same row many times, orders other than the rows'."""
    V = 1003
    for shift in range(0, 9):
        for ld in (V, V + 5, 1024):
            flat = torch.randn(7 * ld + 16, device="cuda").mul_(3).to(dtype)
            x = flat[shift:].as_strided((6, V), (ld, 1))
            y = torch.randint(0, V, (6,), device="cuda")
            _check_fwd(x, y, 9)
            _check_bwd(x, y, 9)
    x, y, _ = _logits(1, V, dtype)
    same = x.expand(5, V)
    out = _check_fwd(same, y.expand(5), 3)
    assert (out.entropy == out.entropy[0]).all()
    box = torch.randn(3, 4, V, device="cuda").to(dtype)
    y = torch.randint(0, V, (4, 3), device="cuda")
    out = token_logprobs(box.transpose(0, 1), y, top_k=2)
    ref = token_logprobs(box.transpose(0, 1).reshape(12, V), y.reshape(12), top_k=2)
    assert torch.equal(out.logprobs.view(-1), ref.logprobs) and torch.equal(out.top_ids.view(12, 2), ref.top_ids)
    cols = torch.randn(V, 6, device="cuda").to(dtype).t()
    _check_fwd(cols.contiguous(), None, 2)
    assert torch.equal(token_logprobs(cols, top_k=2).top_ids, token_logprobs(cols.contiguous(), top_k=2).top_ids)


def test_offsets_beyond_32_bits():
    """Rows more than 2^31 elements apart, gradient included."""
    V, ld = 4099, (1 << 31) + 4104
    flat = torch.zeros(ld + V, device="cuda", dtype=torch.bfloat16)
    x = flat.as_strided((2, V), (ld, 1))
    x.copy_(torch.randn(2, V, device="cuda"))
    y = torch.tensor([3, V - 1], device="cuda")
    _check_fwd(x, y, 4)
    values, ids = token_logprobs(x, top_k=4)[2:]
    out = torch.empty(2, V, device="cuda", dtype=torch.bfloat16)
    ref, grad, off, grad_off = oracle.distill(x, values, ids, 1.5, "bucket")
    loss = distill_topk_fwd_bwd_(x, values, ids, 1.0, tail="bucket", temperature=1.5, out=out)
    oracle.check(loss, ref, off, "loss")
    oracle.check(out, grad, grad_off, "gradient")
    a = x.detach().requires_grad_(True)
    (got,) = torch.autograd.grad(distill_topk(a, values, ids, tail="bucket", temperature=1.5).sum(), a)
    oracle.check(got, grad, grad_off, "gradient of the autograd form")
    _check_bwd(x, y, 4)
    distill_topk_fwd_bwd_(x, values, ids, 1.0, tail="bucket", temperature=1.5)
    assert torch.equal(x, out) and not flat[V:ld].any()


def test_many_rows():
    """More rows than a grid dimension of 65535, a vocabulary of a few columns."""
    x, y, _ = _logits(70001, 9, torch.float32)
    _check_fwd(x, y, 3)
    _check_bwd(x, y, 3)


# ------------------------------------------------------------------------------------------------


def _teacher(x, K, gen, t=1.0, dtype=torch.float32):
    z = (x.float() + torch.randn(x.shape, generator=gen, device="cuda")) / t
    z = torch.nan_to_num(z, nan=0.0, neginf=-30.0)
    values, ids = torch.log_softmax(z, 1).topk(K)
    return values.to(dtype), ids


def _check_distill(x, values, ids, t, tail, scale=0.5):
    ref, grad, off, grad_off = oracle.distill(x, values, ids, t, tail)
    out = torch.full_like(x, 77.0)
    loss = distill_topk_fwd_bwd_(x, values, ids, scale, temperature=t, tail=tail, out=out)
    oracle.check(loss, ref, off, "loss")
    oracle.check(out, grad * scale, grad_off * scale, "gradient")
    a = x.detach().requires_grad_(True)
    w = torch.rand(x.shape[0], device="cuda") + 0.5
    loss2 = distill_topk(a, values, ids, temperature=t, tail=tail)
    oracle.check(loss2, ref, off, "loss of the autograd form")
    (got,) = torch.autograd.grad(loss2, a, w)
    w = w.cpu().double()[:, None]
    oracle.check(got, grad * w, grad_off * w, "gradient of the autograd form")
    b = x.detach().clone()
    loss3 = distill_topk_fwd_bwd_(b, values, ids, scale, temperature=t, tail=tail)
    assert torch.equal(loss3, loss) and torch.equal(b, out), "in place"


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,K", [(1, 1, 1), (3, 2, 2), (4, 7, 3), (5, 128, 128), (3, 1000, 17), (300, 513, 8), (2, 8191, 128),
                                   (3, 50257, 64), (1, 128256, 128), (2, 151937, 33), (1, 262147, 5)])
def test_distill_values_and_gradient(tail, dtype, T, V, K):
    x, _, gen = _logits(T, V, dtype, seed=V)
    for t, value_type in ((1.0, torch.float32), (2.0, torch.bfloat16)):
        values, ids = _teacher(x, K, gen, t, value_type)
        if T > 2:
            ids[1] = -1
            ids[2, K // 2:] = -1 if K > 1 else ids[2, K // 2:]
        _check_distill(x, values, ids if t == 1.0 else ids.int(), t, tail)
    _check_distill(x, values.half(), ids, 0.5, tail)


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_rows_that_stand_for_nothing(tail, dtype):
    V, K = 9000, 6
    x, _, gen = _logits(12, V, dtype, seed=9)
    values, ids = _teacher(x, K, gen)
    low = torch.finfo(dtype).min
    x[0] = float("nan")                                # left out: not looked at
    ids[0] = -1
    ids[1, 1:] = V + 5                                 # out of range: absent, whatever the value
    values[1, 1:] = float("nan")
    ids[2, 3] = ids[2, 0]                              # named twice, and three times
    ids[2, 4] = ids[2, 0]
    x[3] = NEG                                         # the student has nothing
    x[4] = NEG                                         # ... nothing but the teacher's tokens
    x[4, ids[4]] = 1.0
    x[5, ids[5, 2]] = NEG                              # ... not one of the teacher's tokens
    values[6] = NEG
    x[7] = low
    x[8] = low
    x[8, ids[8]] = 2.0
    values[9] = torch.log_softmax(torch.tensor([40.0, 0, 0, 0, 0, 0], device="cuda"), 0)
    x[10, ids[10]] = 30.0                              # next to nothing outside
    x[11] = NEG
    x[11, :50] = 0.5
    _check_distill(x, values, ids, 1.0, tail)
    _check_distill(x, values, ids, 0.7, tail)
    bad = x[10:].clone()
    bad[0, 17] = float("nan")
    bad[1, 17] = float("inf")
    out = torch.empty_like(bad)
    loss = distill_topk_fwd_bwd_(bad, values[10:], ids[10:], 1.0, tail=tail, out=out)
    assert loss.isnan().all() and out.isnan().all()


def test_distill_views_leave_their_surroundings_alone():
    for dtype in DTYPES:
        for shift in (0, 1, 3):
            V, T, K = 1001, 5, 12
            big = torch.full((T + 2, V + 29), 7.0, device="cuda", dtype=dtype)
            x, _, gen = _logits(T, V, dtype, seed=2)
            values, ids = _teacher(x, K, gen)
            ids[3] = -1
            # rows at other addresses are summed up in another order: each result is held to the 64-bit form
            ref, grad, off, grad_off = oracle.distill(x, values, ids, 1.0, "bucket")
            view = big[1:-1, 8 + shift: 8 + shift + V]
            oracle.check(distill_topk_fwd_bwd_(x, values, ids, 1.0, tail="bucket", out=view), ref, off, "loss")
            oracle.check(view, grad, grad_off, "out elsewhere")
            view.copy_(x)
            oracle.check(distill_topk_fwd_bwd_(view, values, ids, 1.0, tail="bucket"), ref, off, "loss")
            oracle.check(view, grad, grad_off, "in place elsewhere")
            keep = torch.ones_like(big, dtype=torch.bool)
            keep[1:-1, 8 + shift: 8 + shift + V] = False
            assert (big[keep] == 7.0).all()


def test_gradients_by_differences():
    """Directional derivative of the kernels' own results. With step e = 2^-6 along a direction of unit-variance
    components a central difference is off by e^2 / 6 of the third derivative (below 30 for these rows of 64 logits) and by the
    results' rounding over e: 30 / 6 * 2^-12 + 2^-17 * 2^6 < 2e-3, against derivatives of order 1."""
    x, y, gen = _logits(1, 64, torch.float32, std=1.0)
    u = torch.randn(1, 64, generator=gen, device="cuda")
    u = u / u.norm()
    values, ids = _teacher(x, 8, gen)
    e = 2.0 ** -6
    forms = [lambda v: token_logprobs(v, y).logprobs, lambda v: token_logprobs(v, y, temperature=0.8).entropy,
             lambda v: token_logprobs(v, y, top_k=2).top_logprobs.sum(1),
             lambda v: distill_topk(v, values, ids, tail="bucket"), lambda v: distill_topk(v, values, ids, temperature=1.5)]
    for i, f in enumerate(forms):
        a = x.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(f(a).sum(), a)
        slope = ((f(x + e * u) - f(x - e * u)) / (2 * e)).item()
        assert abs(slope - float((g * u).sum())) < 2e-3, i


def test_results_repeat_bit_for_bit():
    x, y, gen = _logits(37, 50257, torch.bfloat16)
    values, ids = _teacher(x, 64, gen)
    first = None
    for _ in range(3):
        out, grad = token_logprobs(x, y, top_k=64), torch.empty_like(x)
        loss = distill_topk_fwd_bwd_(x, values, ids, 1.0, tail="bucket", out=grad)
        now = [*out, loss, grad]
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


def test_captured_and_replayed():
    """Forward, gradient and the fused form in one graph, replayed on other contents; a second graph beside it."""
    T, V, K = 33, 4099, 8
    x, y, gen = _logits(T, V, torch.bfloat16)
    values, ids = _teacher(x, K, gen)
    gl, gh = torch.randn(T, generator=gen, device="cuda"), torch.randn(T, generator=gen, device="cuda")
    grad = torch.empty_like(x)

    def once():
        a = x.detach().requires_grad_(True)
        out = token_logprobs(a, y, top_k=K)
        (g,) = torch.autograd.grad([out.logprobs, out.entropy], a, [gl, gh])
        loss = distill_topk_fwd_bwd_(x, values, ids, 1.0, tail="bucket", out=grad)
        return [out.logprobs.detach(), out.top_logprobs.detach(), out.top_ids, g, loss, grad]

    once()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = once()
        graphs.append((graph, kept))
    for seed in (1, 2):
        x2, y2, _ = _logits(T, V, torch.bfloat16, seed=seed)
        x.copy_(x2)
        y.copy_(y2)
        y[seed] = -100
        ref = [t.clone() for t in once()]
        for graph, kept in graphs:
            grad.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(kept, ref))


def test_streams_at_once():
    cases = []
    for seed in range(3):
        x, y, gen = _logits(64, 32000, torch.bfloat16, seed=seed)
        values, ids = _teacher(x, 16, gen)
        ref_grad = torch.empty_like(x)
        cases.append((x, y, values, ids, token_logprobs(x, y, top_k=16),
                      distill_topk_fwd_bwd_(x, values, ids, 1.0, out=ref_grad), ref_grad))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(5):
        for s, (x, y, values, ids, *_) in zip(streams, cases):
            with torch.cuda.stream(s):
                grad = torch.empty_like(x)
                got.append((token_logprobs(x, y, top_k=16), distill_topk_fwd_bwd_(x, values, ids, 1.0, out=grad), grad))
    torch.cuda.synchronize()
    for i, (out, loss, grad) in enumerate(got):
        ref = cases[i % 3]
        assert all(torch.equal(a, b) for a, b in zip(out, ref[4])) and torch.equal(loss, ref[5]) and torch.equal(grad, ref[6])


def test_no_rows():
    x = torch.zeros(0, 100, device="cuda", dtype=torch.bfloat16)
    out = token_logprobs(x, torch.zeros(0, device="cuda", dtype=torch.int64), top_k=3)
    assert out.logprobs.shape == (0,) and out.top_ids.shape == (0, 3)
    ids = torch.zeros(0, 4, device="cuda", dtype=torch.int64)
    assert distill_topk_fwd_bwd_(x, torch.zeros(0, 4, device="cuda"), ids, 1.0).shape == (0,)
    a = x.float().requires_grad_(True)
    distill_topk(a, torch.zeros(0, 4, device="cuda"), ids).sum().backward()
    assert a.grad.shape == (0, 100)


def test_refusals():
    x, y, _ = _logits(4, 100, torch.bfloat16)
    ids, v = torch.zeros(4, 2, device="cuda", dtype=torch.int64), torch.zeros(4, 2, device="cuda")
    with pytest.raises(TypeError):
        token_logprobs(x.double(), y)
    with pytest.raises(ValueError):
        token_logprobs(x, y.cpu())
    with pytest.raises(ValueError):
        distill_topk(x, v, ids.cpu())
    with pytest.raises(ValueError):
        distill_topk(x, v.cpu(), ids)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(1, 1, device="cuda").expand(1, MAX_VOCAB + 1), None)
    with pytest.raises(RuntimeError):    # rows that share memory cannot be written
        distill_topk_fwd_bwd_(x[:1].expand(4, 100), v, ids, 1.0)
    with pytest.raises(RuntimeError):    # nor a gradient that lies across the logits
        distill_topk_fwd_bwd_(x[:3], v[:3], ids[:3], 1.0, out=x[1:])
    C = _ext.C()
    f = torch.zeros(4, device="cuda")
    for bad in (lambda: C.token_logprobs_fwd(x, y, f, f[:3], torch.zeros(4, 2, device="cuda"), None, None, 1.0),
                lambda: C.token_logprobs_fwd(x, y, None, f, torch.zeros(4, 2, device="cuda"), None, None, 1.0),
                lambda: C.token_logprobs_fwd(x, y, f, f, torch.zeros(4, device="cuda"), None, None, 1.0),
                lambda: C.distill_topk(x, v, ids, f, None, None, None, 1.0, 1.0, False),
                lambda: C.distill_topk(x, v[:2], ids, f, None, None, x, 1.0, 1.0, False)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("V,rows", [(600, 700), (50257, 90), (128256, 40)])
def test_distill_runs_of_rows_that_are_left_out(V, rows):
    """Rows without entries alone, in runs and at the ends, between others: what is known ahead of a row must not wait for it."""
    x, _, gen = _logits(rows, V, torch.bfloat16, seed=4)
    values, ids = _teacher(x, 5, gen)
    ref_grad = torch.empty_like(x)
    ref = distill_topk_fwd_bwd_(x, values, ids, 1.0, tail="bucket", out=ref_grad)
    keep = torch.rand(rows, generator=gen, device="cuda") < 0.3
    keep[:7] = False
    keep[rows // 2: rows // 2 + 20] = False
    keep[-9:] = False
    for mask in (keep, ~keep, torch.zeros_like(keep)):
        some = ids.masked_fill(~mask[:, None], -1)
        out = torch.full_like(x, 5.0)
        loss = distill_topk_fwd_bwd_(x, values, some, 1.0, tail="bucket", out=out)
        _ext.check_status()
        assert torch.equal(loss, ref.masked_fill(~mask, 0.0))
        assert torch.equal(out, ref_grad.masked_fill(~mask[:, None], 0.0))


def test_gradients_of_gradients_are_refused():
    x, y, gen = _logits(3, 50, torch.float32)
    values, ids = _teacher(x, 4, gen)
    for f in (lambda v: token_logprobs(v, y).entropy, lambda v: distill_topk(v, values, ids)):
        a = x.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(f(a).sum(), a, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), a)


def test_logits_changed_before_the_backward_are_noticed():
    x, y, _ = _logits(3, 50, torch.float32)
    a = x.clone().requires_grad_(True)
    b = a * 1.0
    loss = token_logprobs(b, y).logprobs.sum()
    b.data.zero_()                     # (not noticed by design of .data)
    b = a * 1.0
    loss = token_logprobs(b, y).logprobs.sum()
    b.mul_(2.0)
    with pytest.raises(RuntimeError):
        loss.backward()


def test_shapes_of_the_autograd_forms():
    x, y, gen = _logits(6, 40, torch.bfloat16)
    values, ids = _teacher(x, 4, gen)
    a = x.view(2, 3, 40).clone().requires_grad_(True)
    out = token_logprobs(a, y.view(2, 3), top_k=2)
    assert out.logprobs.shape == out.entropy.shape == (2, 3) and out.top_ids.shape == (2, 3, 2)
    loss = distill_topk(a, values.view(2, 3, 4), ids.view(2, 3, 4))
    assert loss.shape == (2, 3)
    (g,) = torch.autograd.grad(out.top_logprobs.sum() + loss.sum(), a)
    assert g.shape == a.shape and g.dtype == a.dtype
    one = token_logprobs(x[0], y[0], top_k=2)
    assert one.logprobs.shape == () and one.top_ids.shape == (2,)
    assert not token_logprobs(x, y).entropy.requires_grad


def _far_rows(V, dtype):
    """Rows around +-10^k: all alike (what a mask leaves), a few steps of the type apart, and among ordinary logits."""
    gen = torch.Generator(device="cuda").manual_seed(17)
    rows = []
    for a in (1e3, -6e4, 9e5, -2e6, 3e7, -1e9, 2e10, -1e10, 1e13, -1e17, 1e20, -1e25, 1e29, -3e30, -2e38):
        if abs(a) > torch.finfo(dtype).max:
            continue
        steps = torch.randint(0, 4, (V,), generator=gen, device="cuda")
        rows.append(torch.full((V,), a, device="cuda", dtype=torch.float64))
        rows.append(a * (1 - steps.double() * torch.finfo(dtype).eps))
        mixed = torch.randn(V, generator=gen, device="cuda", dtype=torch.float64) * 3
        rows.append(torch.where(steps == 0, -abs(a), mixed))
        rows.append(torch.where(torch.arange(V, device="cuda") == V // 2, abs(a), mixed))
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5, 257, 50257])
@pytest.mark.parametrize("t", [1.0, 1e-4, 300.0])
def test_logits_far_from_zero(dtype, V, t):
    x = _far_rows(V, dtype)
    y = torch.arange(x.shape[0], device="cuda") % V
    _check_fwd(x, y, min(V, 9), t)
    _check_fwd(x, y, 0, t)
    _check_bwd(x, y, min(V, 9), t)
    _check_bwd(x, y, 0, t, ("lp",))


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5, 257, 50257])
@pytest.mark.parametrize("t", [1.0, 1e-4, 300.0])
def test_distill_logits_far_from_zero(tail, dtype, V, t):
    x = _far_rows(V, dtype)
    T, K = x.shape[0], 4
    gen = torch.Generator(device="cuda").manual_seed(18)
    values = torch.log_softmax(torch.randn(T, K + 1, generator=gen, device="cuda"), 1)[:, :K].contiguous()
    ids = (torch.randint(0, V, (T, 1), generator=gen, device="cuda") + torch.arange(K, device="cuda")) % V
    ref, grad, off, grad_off = oracle.distill(x, values, ids, t, tail)
    a = x.clone().requires_grad_(True)
    loss = distill_topk(a, values, ids, temperature=t, tail=tail)
    oracle.check(loss, ref, off, "loss")
    (got,) = torch.autograd.grad(loss.sum(), a)
    oracle.check(got, grad, grad_off, "gradient")
    got = torch.empty_like(x)
    oracle.check(distill_topk_fwd_bwd_(x, values, ids, 1.0, temperature=t, tail=tail, out=got), ref, off, "loss")
    oracle.check(got, grad, grad_off, "gradient")


def test_logits_overwritten_before_the_backward_are_noticed():
    x, y, _ = _logits(4, 100, torch.float32)
    x.requires_grad_(True)
    z = x * 1.0
    out = token_logprobs(z, y)
    distill_topk_fwd_bwd_(z.detach(), torch.zeros(4, 1, device="cuda"), y[:, None], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.logprobs.sum().backward()


@pytest.mark.parametrize("V", [15000, 20000, 22800, 23100, 23500, 24000, 24570, 25000, 26000, 27000, 28000, 33000, 47000])
def test_vocabularies_around_the_sizes_of_shared_memory(V):
    x, y, gen = _logits(800, V, torch.bfloat16, seed=V)
    values, ids = _teacher(x, 5, gen)
    out = torch.empty_like(x)
    loss = distill_topk_fwd_bwd_(x, values, ids, 1.0, out=out)
    few = slice(797, 800)
    ref, grad, off, grad_off = oracle.distill(x[few], values[few], ids[few], 1.0, "renormalize")
    oracle.check(loss[few], ref, off, "loss")
    oracle.check(out[few], grad, grad_off, "gradient")
    for dtype, K in ((torch.bfloat16, 3), (torch.float32, 128)):
        _check_fwd(x[:200].to(dtype), y[:200], K)
    del x, out
    x, y, _ = _logits(3, 5 * V, torch.bfloat16, seed=V)
    _check_fwd(x, y, 9)


def test_the_extension_refuses_what_the_cpu_form_does():
    x, y, _ = _logits(3, 20, torch.float32)
    ids, v = torch.zeros(3, 2, device="cuda", dtype=torch.int64), torch.zeros(3, 2, device="cuda")
    for device in ("cpu", "cuda"):
        x, y, ids, v = x.to(device), y.to(device), ids.to(device), v.to(device)
        wide = torch.zeros(3, 129, device=device)
        for error, bad in (
                (ValueError, lambda: token_logprobs(x, y, top_k=21)), (ValueError, lambda: token_logprobs(x, y, top_k=-1)),
                (ValueError, lambda: token_logprobs(x, y, temperature=0.0)),
                (ValueError, lambda: token_logprobs(x, y, temperature=math.nan)),
                (ValueError, lambda: token_logprobs(x, y, temperature=math.inf)),
                (ValueError, lambda: token_logprobs(x, y, ignore_index=5)),
                (ValueError, lambda: token_logprobs(wide.repeat(1, 2), top_k=129)),
                (ValueError, lambda: token_logprobs(x, y[:2])), (ValueError, lambda: token_logprobs(x, y[:, None])),
                (TypeError, lambda: token_logprobs(x, y.float())), (TypeError, lambda: token_logprobs(x.long(), y)),
                (ValueError, lambda: token_logprobs(x[:, :0])), (ValueError, lambda: token_logprobs(x[0, 0])),
                (ValueError, lambda: distill_topk(x, v, ids, tail="drop")), (ValueError, lambda: distill_topk(x, v[:, :1], ids)),
                (ValueError, lambda: distill_topk(x, v[:2], ids[:2])), (ValueError, lambda: distill_topk(x, v, ids, temperature=-1.0)),
                (ValueError, lambda: distill_topk(x, v[:, :0], ids[:, :0])), (ValueError, lambda: distill_topk(x, wide, wide.long())),
                (ValueError, lambda: distill_topk(x, v.clone().requires_grad_(True), ids)),
                (ValueError, lambda: distill_topk(x, v[0], ids[0])), (ValueError, lambda: distill_topk(x[0], v, ids)),
                (TypeError, lambda: distill_topk(x, v, ids.float())), (TypeError, lambda: distill_topk(x, v.long(), ids)),
                (ValueError, lambda: distill_topk_fwd_bwd_(x, v, ids, 1.0, out=torch.zeros(3, 21, device=device))),
                (ValueError, lambda: distill_topk_fwd_bwd_(x, v, ids, 1.0, out=x.bfloat16())),
                (ValueError, lambda: distill_topk_fwd_bwd_(x.t(), wide[:1, :2].expand(20, 2), torch.zeros(20, 2, device=device).long(), 1.0)),
                (ValueError, lambda: distill_topk_fwd_bwd_(x[None], v[None], ids[None], 1.0)),
                (ValueError, lambda: distill_topk_fwd_bwd_(x, v, ids, 1.0, temperature=1e5)),
                (ValueError, lambda: distill_topk_fwd_bwd_(x, v, ids, 1.0, tail="")),
                (ValueError, lambda: distill_topk_fwd_bwd_(x, v, ids[:, :1], 1.0))):
            with pytest.raises(error):
                bad()


def test_scoring_without_gradients_is_scoring_with_them():
    x, y, _ = _logits(5, 1000, torch.bfloat16)
    y[3] = -100
    with_grad = token_logprobs(x.clone().requires_grad_(True), y, top_k=4)
    with torch.inference_mode():
        z = x.clone()
        without = token_logprobs(z, y, top_k=4)
        distill_topk_fwd_bwd_(z, without.top_logprobs, without.top_ids, 1.0)
    for a, b in zip(with_grad, without):
        assert torch.equal(a, b)


def test_gradients_that_lie_across_other_arguments_are_refused():
    buffer = torch.zeros(4, 120, device="cuda")
    x, y = torch.randn(4, 100, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.int64)
    ids = torch.arange(8, device="cuda").view(4, 2)
    flat = buffer.view(-1)
    with pytest.raises(RuntimeError, match="values"):
        distill_topk_fwd_bwd_(x, flat[200:208].view(4, 2), ids, 1.0, out=buffer[:, :100])
    with pytest.raises(RuntimeError, match="ids"):
        distill_topk_fwd_bwd_(x, torch.zeros(4, 2, device="cuda"), flat[:8].view(torch.int32).view(4, 2), 1.0, out=buffer[:, :100])
    out, stats = ops.token_logprobs_fwd(x, y, 2, 1.0)
    with pytest.raises(RuntimeError, match="d_entropy"):
        ops.token_logprobs_bwd(x, y, out, stats, None, flat[101:105], None, 1.0, buffer[:, 20:])
    # beside one another is fine
    distill_topk_fwd_bwd_(x, flat[470:478].view(4, 2), ids, 1.0, out=buffer.view(-1)[:400].view(4, 100))


def test_small_results_are_tensors_of_their_own():
    x, y, _ = _logits(3, 50, torch.bfloat16)
    first = token_logprobs(x, y, top_k=2)
    kept = [t.clone() for t in first]
    second = token_logprobs(x.flip(1), y, top_k=2)
    assert all(torch.equal(a, b) for a, b in zip(first, kept))
    second.logprobs.fill_(5.0)
    second.top_ids.zero_()
    assert bool((second.entropy != 5.0).all()) and bool((second.top_logprobs != 0.0).any())
    for t in (*first, *second):
        assert t.is_contiguous() and t.data_ptr() % 16 == 0 and t._base is None
    a = x.clone().requires_grad_(True)
    out = token_logprobs(a, y, top_k=2)
    with torch.no_grad():
        out.top_ids[0, 0] += 0                      # what the backward has kept: noticed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.logprobs.sum().backward()
    out = token_logprobs(a, y, top_k=2)
    out.logprobs.detach().zero_()                   # what it has not: nothing to it
    (out.entropy.sum() + out.logprobs.sum()).backward()
    want, off = oracle.logprobs_grad(x, y, 0, 1.0, torch.ones(3, device="cuda"), torch.ones(3, device="cuda"), None)
    oracle.check(a.grad, want, off, "gradient")
