"""Log probabilities of tokens, entropies, top alternatives and their backward pass, against 64 bits.

Tolerances, fixed before the first run.  With t the distance of a logit from its row's maximum (in log2 units), fp32 rounds
t log2 e and the exponential's argument to 2^-24 |t| each and 2^t to 2^-22; a thread adds at most V / 32 terms, then 10
levels of pairs: with weights p the sums l and w are off by less than 2^-22 (4 + max over p-weighted |t|) + V / 32 2^-24 of
their size in the worst case, in practice by its square root.  Log probabilities (|t| up to ~40 here) and entropies are held
to 4e-6 (1 + |value|), which is 2^-22 times about 17.  The gradient is a product of three such numbers, rounded once: eps / 2
of itself, 1e-5 (|g| + |h| (1 + log V)) p, and for fp16 half of its smallest step, 2^-25.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

import double_attention_b200 as da

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _logits(rows: int, v: int, dtype, seed: int = 0, scale: float = 3.0) -> tuple[torch.Tensor, torch.Tensor]:
    g = torch.Generator("cuda").manual_seed(seed)
    x = (scale * torch.randn(rows, v, device="cuda", generator=g)).to(dtype)
    return x, torch.randint(0, v, (rows,), device="cuda", generator=g)


def _expected(x: torch.Tensor, tokens: torch.Tensor):
    lp = torch.log_softmax(x.double(), -1)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(lp)).sum(-1)
    entropy = torch.where(lp.isnan().any(-1), torch.full_like(entropy, math.nan), entropy)
    return lp, entropy


def _check(x: torch.Tensor, tokens: torch.Tensor, top: int) -> None:
    made = da.token_log_probs(x, tokens, top=top)
    lp, entropy = _expected(x, tokens)
    want = lp.gather(-1, tokens[..., None])[..., 0]
    assert made.log_probs.dtype == made.entropy.dtype == FP32
    for got, value in ((made.log_probs, want), (made.entropy, entropy)):
        assert torch.equal(got.isnan(), value.isnan())
        ok = (got.double() - value).abs() <= 4e-6 * (1 + value.abs())
        # (a value past fp32's range, as -6.8e38 below the largest logit, rounds to an infinity of it)
        assert (ok | value.isnan() | (got == value.float())).all(), (got.double() - value).abs().nan_to_num().max()
    if not top:
        assert made.top_log_probs is None and made.top_tokens is None
        return
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top]
    assert torch.equal(made.top_tokens, order)
    best = lp.gather(-1, order)
    ok = (made.top_log_probs.double() - best).abs() <= 4e-6 * (1 + best.abs())
    assert (ok | best.isnan() | (made.top_log_probs == best.float())).all()


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize(("rows", "v", "top"), [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 31, 31), (4, 33, 32), (1, 2048, 5),
                                                (7, 2047, 0), (64, 50021, 20), (1, 130001, 32), (2, 8193, 1), (1000, 512, 8),
                                                (700, 1001, 32), (600, 8192, 3), (601, 17, 17), (2500, 63, 0), (3, 8200, 32)])
def test_scores(rows, v, top, dtype) -> None:
    _check(*_logits(rows, v, dtype), top)


@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_rows_that_are_hard_to_rank(rows, dtype) -> None:
    v = 3001
    up = torch.linspace(-30, 30, v, device="cuda").to(dtype)
    cases = [up.expand(rows, v), up.flip(0).expand(rows, v), torch.zeros(rows, v, device="cuda", dtype=dtype),
             torch.full((rows, v), -1e4, device="cuda", dtype=dtype),
             (torch.arange(v, device="cuda") % 3).to(dtype).expand(rows, v) * -0.0]
    blocks = torch.full((rows, v), -5.0, device="cuda", dtype=dtype)
    blocks[:, 1000:1040] = 7.0  # the largest lie side by side, all alike
    for x in (*cases, blocks):
        _check(x.contiguous(), torch.arange(rows, device="cuda") % v, 32)


@pytest.mark.parametrize(("rows", "v"), [(2000, 3001), (40, 3001), (40, 20001), (400, 20001), (3, 257), (20, 1999)])
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("top", [1, 9, 32])
def test_alternatives_by_few_and_by_many_threads_a_row(rows, v, top, dtype) -> None:
    x, tokens = _logits(rows, v, dtype, 21)
    _check(x, tokens, top)
    x[:, v // 3: v // 3 + 200] = 20.0   # more equal ones than the top, side by side
    x[1::2, 5] = 21.0
    _check(x, tokens, top)
    x[:, ::2] = -math.inf
    x[0, 1:] = -math.inf                 # fewer numbers than the top
    x[0, 1] = 1.0
    tokens[:] = 1
    _check(x, tokens, top)
    x[:, 7::11] = math.nan
    made = da.token_log_probs(x, tokens, top=top)
    want = torch.arange(7, v, 11, device="cuda")[:top]
    assert torch.equal(made.top_tokens[:, :len(want)], want.expand(rows, -1)) and made.entropy.isnan().all()


@pytest.mark.parametrize("rows", [6, 900])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_infinities_and_nan(rows, dtype) -> None:
    x, tokens = _logits(rows, 1003, dtype, 1)
    x[:, ::3] = -math.inf
    tokens[1] = 0                    # a token that is ruled out: minus infinity
    x[2] = -math.inf                 # nothing left
    x[3] = -math.inf
    x[3, 77], tokens[3] = 2.0, 77    # one left
    x[4, 500] = math.nan
    x[5, 10] = math.inf
    _check(x, tokens, 0)
    made = da.token_log_probs(x, tokens, top=20)
    assert made.log_probs[1] == -math.inf and made.log_probs[3] == 0 and made.entropy[3] == 0
    assert made.log_probs[[2, 4, 5]].isnan().all() and made.entropy[[2, 4, 5]].isnan().all()
    assert made.top_tokens[4, 0] == 500 and made.top_tokens[5, 0] == 10
    assert torch.equal(made.top_tokens[2], torch.arange(20, device="cuda"))
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[[2, 4, 5]] = False
    _check(x[keep], tokens[keep], 20)


@pytest.mark.parametrize("rows", [5, 800])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_masks_of_the_lowest_value(rows, dtype) -> None:
    x, tokens = _logits(rows, 1500, dtype, 12)
    low = torch.finfo(dtype).min
    x[:, 1::2] = low
    x[1] = low                        # nothing else: an even row
    x[2] = low
    x[2, ::3] = -math.inf             # an even row of two thirds
    tokens[2] = 1
    x[3, 0] = torch.finfo(dtype).max
    _check(x, tokens, 30)
    g = torch.ones(rows, device="cuda")
    d = _gradient(x, tokens, g, g)
    assert d.isfinite().all() and not d[2, ::3].any()
    even = -1.0 / 1500
    token = torch.zeros(1500, device="cuda").index_fill_(0, tokens[1], 1.0)
    assert ((d[1].double() - token - even).abs() <= torch.finfo(dtype).eps + 1e-5).all()


def test_logits_far_from_zero() -> None:
    x, tokens = _logits(5, 5000, FP32, 2)
    _check(x + 30000.0, tokens, 4)
    _check(x - 30000.0, tokens, 4)
    spread, tokens = _logits(5, 5000, FP32, 3, 2000.0)
    _check(spread, tokens, 4)


def test_strides_shapes_and_token_types() -> None:
    x, tokens = _logits(24, 1000, BF16, 4)
    want = da.token_log_probs(x, tokens, top=3)
    wide = torch.zeros(24, 1011, dtype=BF16, device="cuda")
    wide[:, 5:1005] = x
    for t in (wide[:, 5:1005], x.t().contiguous().t()):
        for got, value in zip(da.token_log_probs(t, tokens.int(), top=3), want):
            assert (got - value).abs().max() <= 4e-6 * (1 + value.abs().max())
    shaped = da.token_log_probs(x.view(2, 3, 4, 1000), tokens.view(2, 3, 4), top=3)
    assert shaped.entropy.shape == (2, 3, 4) and torch.equal(shaped.top_tokens.view(24, 3), want.top_tokens)
    one = da.token_log_probs(x[0], tokens[0], top=3)
    assert one.log_probs.shape == () and one.top_tokens.shape == (3,)
    none = da.token_log_probs(x[:0], tokens[:0], top=3)
    assert none.log_probs.shape == (0,) and none.top_tokens.shape == (0, 3)


def _gradient(x, tokens, g, h):
    x = x.clone().requires_grad_()
    made = da.token_log_probs(x, tokens)
    outs = [(o, d) for o, d in ((made.log_probs, g), (made.entropy, h)) if d is not None]
    return torch.autograd.grad([o for o, _ in outs], x, [d for _, d in outs])[0]


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize(("rows", "v"), [(1, 1), (3, 7), (5, 2048), (64, 50021), (1000, 513), (2, 4099), (700, 2047)])
@pytest.mark.parametrize("which", ["log_probs", "entropy", "both"])
def test_gradient(rows, v, dtype, which) -> None:
    x, tokens = _logits(rows, v, dtype, 5)
    if v > 3:
        x[:, 2] = -math.inf
        tokens = torch.where(tokens == 2, 1, tokens)
    gen = torch.Generator("cuda").manual_seed(6)
    g = torch.randn(rows, device="cuda", generator=gen) if which != "entropy" else None
    h = torch.randn(rows, device="cuda", generator=gen) if which != "log_probs" else None
    got = _gradient(x, tokens, g, h)
    x64 = x.double().requires_grad_()
    lp = torch.log_softmax(x64, -1)
    p = lp.exp()
    loss = 0.0
    if g is not None:
        loss = loss + (lp.gather(1, tokens[:, None])[:, 0] * g.double()).sum()
    if h is not None:
        loss = loss - (torch.where(p > 0, p * lp.clamp_min(-1e30), torch.zeros_like(p)).sum(1) * h.double()).sum()
    want, = torch.autograd.grad(loss, x64)
    want = torch.where(x.isneginf(), torch.zeros_like(want), want)
    assert got.dtype == dtype and got.shape == x.shape
    size = sum(d.double().abs()[:, None] * f for d, f in ((g, 1.0), (h, 1.0 + math.log(v))) if d is not None)
    token = torch.zeros_like(p).scatter_(1, tokens[:, None], 1.0)
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 1e-5 * size * (p + 1e-1 * token) + (2.0**-25 if dtype == FP16 else 1e-30)
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() - bound).max()
    assert not got[x.isneginf()].any()


def test_gradient_of_strided_logits() -> None:
    x, tokens = _logits(37, 1000, BF16, 13)
    g = torch.randn(37, device="cuda")
    want = _gradient(x, tokens, g, g)
    wide = torch.zeros(37, 1011, dtype=BF16, device="cuda")
    wide[:, 5:1005] = x
    for t in (wide.requires_grad_(), x.t().contiguous().requires_grad_()):
        view = t[:, 5:1005] if t.shape[1] == 1011 else t.t()
        made = da.token_log_probs(view, tokens.int())
        d, = torch.autograd.grad((made.log_probs, made.entropy), t, (g, g))
        d = d[:, 5:1005] if t.shape[1] == 1011 else d.t()
        # (sums in another order: both sides round, half a step, 2^-8, each)
        assert ((d.float() - want.float()).abs() <= 2.0**-7 * want.float().abs() + 1e-6).all()


def test_gradient_against_differences() -> None:
    x, tokens = _logits(4, 300, FP32, 7)
    g, h = torch.tensor([1.0, -2.0, 0.5, 1.5], device="cuda"), torch.tensor([0.3, 0.0, -1.0, 2.0], device="cuda")
    got = _gradient(x, tokens, g, h)

    def loss(z):
        lp, entropy = _expected(z, tokens)
        return lp.gather(1, tokens[:, None])[:, 0] * g.double() + entropy * h.double()

    step = 1e-5
    for column in (0, 17, 123, 299, int(tokens[0])):
        up, down = x.double(), x.double()
        up[:, column] += step
        down[:, column] -= step
        slope = (loss(up) - loss(down)) / (2 * step)
        assert ((got[:, column].double() - slope).abs() <= 2e-5).all()


def test_tokens_that_are_none_and_tokens_outside() -> None:
    x, tokens = _logits(6, 100, BF16, 8)
    tokens[0], tokens[1], tokens[2] = -100, 100, -1
    x.requires_grad_()
    made = da.token_log_probs(x, tokens)
    assert made.log_probs[0] == 0 and made.log_probs[1:3].isnan().all() and made.log_probs[3:].isfinite().all()
    assert made.entropy.isfinite().all()
    made.entropy.sum().backward(retain_graph=True)
    assert x.grad.isfinite().all()
    x.grad = None
    made.log_probs[[0, 3, 4, 5]].sum().backward()
    assert not x.grad[0].any() and x.grad[3:].isfinite().all()


def test_alternatives_carry_no_gradient_and_cross_entropy_agrees() -> None:
    x, tokens = _logits(300, 2048, FP32, 9)
    x.requires_grad_()
    made = da.token_log_probs(x, tokens, top=4)
    assert not made.top_log_probs.requires_grad and not made.top_tokens.requires_grad
    loss = -made.log_probs.mean()
    loss.backward()
    mine, x.grad = x.grad, None
    other = F.cross_entropy(x, tokens)
    other.backward()
    assert abs(loss.item() - other.item()) <= 4e-6 * (1 + other.item())
    assert ((mine - x.grad).abs() <= 1e-5 / 300).all()


def test_captured_and_on_another_stream() -> None:
    x, tokens = _logits(40, 3001, BF16, 10)
    x.requires_grad_()
    g = torch.ones(40, device="cuda")
    want = da.token_log_probs(x, tokens)
    want_d, = torch.autograd.grad(want.log_probs, x, g)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        made = da.token_log_probs(x, tokens)
        d, = torch.autograd.grad(made.log_probs, x, g)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(made.entropy, want.entropy) and torch.equal(d, want_d)
    del made, want
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        captured = da.token_log_probs(x, tokens, top=5)
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    graph.replay()
    with torch.no_grad():
        for got, value in zip(captured, da.token_log_probs(x, tokens, top=5)):
            assert torch.equal(got, value)


def test_a_training_step_in_a_graph() -> None:
    x, tokens = _logits(40, 1001, BF16, 12)
    g, h = torch.randn(40, device="cuda"), torch.randn(40, device="cuda")
    x.requires_grad_()

    def step():
        made = da.token_log_probs(x, tokens)
        return torch.autograd.grad((made.log_probs, made.entropy), x, (g, h))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (13, 14):
        with torch.no_grad():
            x.copy_(_logits(40, 1001, BF16, seed)[0])
        graph.replay()
        assert torch.equal(captured, step())


def test_ways_to_the_gradient() -> None:
    """One gradient however it is asked for: of several uses, of an expanded one, of tokens in 32 bits, of strided
    logits, under saved-tensor hooks; and the graph's own checks of what was kept."""
    x, tokens = _logits(24, 500, FP32, 15)
    x.requires_grad_()
    made = da.token_log_probs(x, tokens)
    want, = torch.autograd.grad(made.log_probs, x, torch.ones(24, device="cuda"), retain_graph=True)
    again, = torch.autograd.grad(made.log_probs.sum(), x, retain_graph=True)
    assert torch.equal(again, want)
    assert torch.equal(torch.autograd.grad(made.log_probs.view(4, 6).t().sum(), x)[0], want)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(made.log_probs.sum(), x)
    assert torch.equal(torch.autograd.grad(da.token_log_probs(x, tokens.int()).log_probs.sum(), x)[0], want)
    wide = torch.zeros(24, 700, device="cuda")
    wide[:, 100:600] = x.detach()
    wide.requires_grad_()
    d, = torch.autograd.grad(da.token_log_probs(wide[:, 100:600], tokens).log_probs.sum(), wide)
    assert torch.equal(d[:, 100:600], want) and not d[:, :100].any() and not d[:, 600:].any()
    with torch.autograd.graph.save_on_cpu():
        made = da.token_log_probs(x, tokens)
    assert torch.equal(torch.autograd.grad(made.log_probs.sum(), x)[0], want)
    made = da.token_log_probs(x, tokens, top=3)
    assert made.log_probs.requires_grad and made.entropy.requires_grad and not made.top_log_probs.requires_grad
    with torch.no_grad():
        assert not da.token_log_probs(x, tokens).entropy.requires_grad
        x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(made.log_probs.sum(), x)


def test_refusals() -> None:
    x, tokens = _logits(4, 50, BF16, 11)
    with pytest.raises(ValueError, match="float32"):
        da.token_log_probs(x.double(), tokens)
    with pytest.raises(ValueError, match="tokens"):
        da.token_log_probs(x, tokens[:3])
    with pytest.raises(ValueError, match="int64"):
        da.token_log_probs(x, tokens.float())
    with pytest.raises(ValueError, match="alternatives"):
        da.token_log_probs(x, tokens, top=33)
    with pytest.raises(ValueError, match="alternatives"):
        da.token_log_probs(x[:, :3], tokens % 3, top=4)
    with pytest.raises(ValueError, match="V at least 1"):
        da.token_log_probs(x[:, :0], tokens)
    with pytest.raises(ValueError, match="one device"):
        da.token_log_probs(x, tokens.cpu())
    with pytest.raises(ValueError, match="CUDA"):
        da.token_log_probs(x.cpu(), tokens.cpu())
    x.requires_grad_()
    d, = torch.autograd.grad(da.token_log_probs(x, tokens).log_probs.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        d.sum().backward()
