"""Vocabulary operators at the ends of their ranges, against 64-bit references."""
import pytest
import torch

import fugatensor_b200 as ft
import fugatensor_b200.nn.functional as F
from fugatensor_b200 import _fgt, _native
from tests import _vocab as R

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "f16", "bf16"]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# --------------------------------------------- cross-entropy, wide rows ----
# Exponentials below 2^-126 of a row's reference are 0 (ex2.approx.ftz), and the sum that they are
# divided by is at least half a reference: a gradient is off by up to 2^-125 of its seed that way.
FLUSHED = 2.0 ** -124


def check_rows(x, t, dtype, eps=0.0):
    """Row losses and gradients, together and the loss alone, with a seed per row."""
    seed = 0.5 + torch.rand(x.shape[0], device="cuda", generator=gen(1))
    # neither changes when a row is shifted; at its largest value the reference loses nothing to lse's size
    shifted = x.double() - x.double().amax(1, keepdim=True)
    loss, _, grad, gbound = R.cross_entropy(shifted, t, eps=eps, reduction="none", seed=seed)
    lbound = R.cross_entropy(x, t, eps=eps, reduction="none")[1]
    X, T = R.wrap(x), R.wrap(t)
    l = F.cross_entropy(X, T, label_smoothing=eps, reduction="none")
    d = ft.grad(l, X, seed=R.wrap(seed))
    ft.evaluate(l, d)
    R.check(l.torch(), loss, lbound + R.U32 * loss.abs(), "loss")
    R.check(d.torch(), grad, R.rounded(gbound + FLUSHED * seed[:, None].double(), grad, dtype), "gradient")
    alone = F.cross_entropy(X, T, label_smoothing=eps, reduction="none").torch()
    R.check(alone, loss, lbound + R.U32 * loss.abs(), "loss alone")


# a warp, a CTA, a cluster per row, and a CTA of 64 threads over many rows; `block` is what the group's
# threads read first: every other block is low, so a thread's reference is far below its later values
@pytest.mark.parametrize("dtype,rows,vocab,block", [
    ("f32", 12, 500, 128), ("f32", 12, 5003, 2048), ("f32", 12, 32001, 2048), ("f32", 4200, 2400, 256),
    ("f16", 12, 500, 256), ("f16", 12, 5003, 2048), ("f16", 12, 50021, 4096),
    ("bf16", 12, 500, 256), ("bf16", 12, 5003, 2048), ("bf16", 12, 50021, 4096)])
@pytest.mark.parametrize("eps", [0.0, 0.1])
@pytest.mark.parametrize("rest", [-5.0, -9.0])
def test_cross_entropy_of_rows_whose_first_values_are_far_below_the_others(dtype, rows, vocab, block, eps, rest):
    g = gen(21)
    depth = torch.tensor([80, 84, 86, 87, 88, 88.5, 89, 90, 91, 92, 95, 100], device="cuda")
    x = torch.randn(rows, vocab, device="cuda", generator=g) * 0.5 + rest
    low = (torch.arange(vocab, device="cuda") // block) % 2 == 0
    x = torch.where(low[None, :], -depth[torch.arange(rows, device="cuda") % 12, None], x)
    x[:, 0] = 0.0
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    check_rows(x.to(R.TORCH[dtype]), t, dtype, eps)


@pytest.mark.parametrize("dtype,vocab", [("f32", 503), ("f32", 5003), ("f16", 5007), ("bf16", 50023)])
@pytest.mark.parametrize("depth", [80.0, 86.0, 88.0, 90.0, 96.0])
def test_cross_entropy_of_rows_whose_last_values_are_far_below_the_others(dtype, vocab, depth):
    """An odd vocabulary that is padded at its end: the single values are a thread's first."""
    g = gen(22)
    x = torch.randn(16, vocab, device="cuda", generator=g)
    x[:, vocab - 3:] = -depth
    t = torch.randint(0, vocab, (16,), device="cuda", generator=g)
    check_rows(x.to(R.TORCH[dtype]), t, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(300, 500), (300, 4096), (300, 5001), (40, 33001)])
@pytest.mark.parametrize("spread", [15.0, 20.0, 25.0, 30.0, 60.0])
def test_cross_entropy_of_widely_spread_rows(dtype, rows, vocab, spread):
    g = gen(23)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * spread).to(R.TORCH[dtype])
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    check_rows(x, t, dtype)


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -20, 2.0 ** -60])
def test_gradient_of_a_mean_over_rows_with_one_value_far_above_the_others(scale):
    """The gradient's factor g / sum is far from f32's limits wherever a thread's reference lies."""
    g = gen(24)
    rows, vocab = 8192, 600
    x = 2.0 * torch.rand(rows, vocab, device="cuda", generator=g)
    at = torch.arange(rows, device="cuda")
    x[at, 300 + at % 290] = 80.0 + (at % 7).float()
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    _, _, grad, gbound = R.cross_entropy(x, t, seed=torch.tensor(scale, device="cuda"))
    X = R.wrap(x)
    got = ft.grad(F.cross_entropy(X, R.wrap(t)) * scale, X).torch()
    R.check(got, grad, R.rounded(gbound + FLUSHED * scale / rows, grad, "f32"))


def test_cross_entropy_of_rows_far_from_zero():
    """References beyond 2^24, where whole numbers are no longer all f32 values."""
    g = gen(25)
    x = torch.randn(24, 5003, device="cuda", generator=g) * 2.0
    x[:, :2048] = -90.0
    x[:, 0] = 0.0
    far = torch.tensor([0.0, 1e3, -1e4, 1e5, 1e6, -3e6, 8e6, 1.3e7, -2e7, 1e8, 1e12, -1e20], device="cuda").repeat(2)
    x += far[:, None]
    t = torch.randint(0, 5003, (24,), device="cuda", generator=g)
    check_rows(x, t, "f32")


@pytest.mark.parametrize("dtype,vocab", [("f32", 515), ("f32", 5003), ("bf16", 600), ("bf16", 40001)])
def test_smoothed_loss_of_columns_at_the_lowest_value(dtype, vocab):
    """(e / vocab) * sum(x) is far inside f32 although sum(x) is not."""
    g = gen(28)
    x = torch.randn(6, vocab, device="cuda", generator=g).to(R.TORCH[dtype])
    x[:, vocab // 3:vocab // 2] = torch.finfo(x.dtype).min
    x[1, vocab - 1] = torch.finfo(x.dtype).min
    t = torch.randint(0, vocab // 3, (6,), device="cuda", generator=g)
    check_rows(x, t, dtype, eps=0.1)


# ------------------------------------------------- cross-entropy, no rows --
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("shape", [(0, 40), (2, 0, 40)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_cross_entropy_without_rows(reduction, shape, dtype):
    X = R.wrap(torch.empty(shape, device="cuda", dtype=R.TORCH[dtype]))
    T = R.wrap(torch.empty(shape[:-1], device="cuda", dtype=torch.int64))

    def make():
        loss = F.cross_entropy(X, T, reduction=reduction)
        seed = R.wrap(torch.ones(shape[:-1], device="cuda")) if reduction == "none" else None
        return loss, ft.grad(loss, X, seed=seed)

    def check_loss(l):
        l = l.torch()
        assert l.shape == (shape[:-1] if reduction == "none" else ()) and not l.any() and l.dtype is torch.float32

    check_loss(make()[0])
    d = make()[1].torch()
    assert d.shape == shape and d.dtype is R.TORCH[dtype]
    l, d = make()
    ft.evaluate(l, d)
    check_loss(l)
    assert d.torch().shape == shape


# ------------------------------------------------ logit rules, many biases --
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("index", ["i32", "i64"])
@pytest.mark.parametrize("rows,vocab,biases", [(3, 40, 513), (2, 5001, 5000), (2, 50021, 40000), (1, 128000, 128000)])
def test_adjust_logits_with_many_biases(dtype, index, rows, vocab, biases):
    """Whole numbers, so that sums are exact in any order; with and without a history and a mask."""
    g = gen(26)
    x = torch.randint(-30, 31, (rows, vocab), device="cuda", generator=g).to(R.TORCH[dtype])
    ids = torch.randint(-2, vocab + 2, (rows, biases), device="cuda", generator=g, dtype=R.TORCH[index])
    ids[:, ::9] = 7  # many for one token
    bias = torch.randint(-2, 3, (rows, biases), device="cuda", generator=g).float()
    tokens = torch.randint(0, vocab, (rows, 700), device="cuda", generator=g, dtype=torch.int32)
    words = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), device="cuda", generator=g, dtype=torch.int32)
    for t, a in ((None, None), (tokens, words)):
        out = F.adjust_logits(R.wrap(x), None if t is None else R.wrap(t), presence=1.0, frequency=2.0, bias_tokens=R.wrap(ids),
                              bias=R.wrap(bias), allowed=None if a is None else R.wrap(a)).torch()
        ref, _ = R.adjust_logits(x, t, presence=1.0, frequency=2.0, bias_tokens=ids, bias=bias, allowed=a)
        assert torch.equal(out, ref.to(out.dtype))


@pytest.mark.parametrize("places", [(0, 1, 2, 3), (0, 31, 32, 33), (5, 700, 1500, 1999), (1, 511, 512, 1024)])
def test_many_biases_of_one_token_add_in_their_order(places):
    """2^24 + 1 + 1 - 2^24 in f32, in order, is 0; any other association gives 2."""
    ids = torch.arange(2000, device="cuda", dtype=torch.int32)[None] % 400 + 100
    bias = torch.zeros(1, 2000, device="cuda")
    for p, b in zip(places, (2.0 ** 24, 1.0, 1.0, -2.0 ** 24)):
        ids[0, p], bias[0, p] = 3, b
    out = F.adjust_logits(R.wrap(torch.zeros(1, 600, device="cuda")), bias_tokens=R.wrap(ids), bias=R.wrap(bias)).torch()
    assert not out.any()


def test_a_million_biases():
    """The work grows with the list, not with its square; all for one token, and spread out."""
    n, vocab = 1 << 20, 128000
    x = torch.zeros(1, vocab, device="cuda")
    bias = torch.ones(1, n, device="cuda")
    one = torch.full((1, n), 77, device="cuda", dtype=torch.int32)
    out = F.adjust_logits(R.wrap(x), bias_tokens=R.wrap(one), bias=R.wrap(bias)).torch()
    assert float(out[0, 77]) == n and float(out.sum()) == n
    each = (torch.arange(n, device="cuda", dtype=torch.int32) % vocab)[None]
    out = F.adjust_logits(R.wrap(x), bias_tokens=R.wrap(each), bias=R.wrap(bias)).torch()
    assert torch.equal(out[0], torch.bincount(each[0].long(), minlength=vocab).float())


# -------------------------------------------------- embedding gradient -----
TIERS = [1024, 8192, 16384, 32768, 65536, 131072, 1 << 18]  # tokens at which the sort takes another form


@pytest.mark.parametrize("n", [m for t in TIERS for m in (t, t + 1)] + [12000, 24000, 200000])
@pytest.mark.parametrize("vocab", [300, 40000, 300000])  # one, two and three passes
@pytest.mark.parametrize("dim", [4, 9])
def test_embedding_grad_in_every_form_of_the_sort(n, vocab, dim):
    """Whole numbers: the sums are exact. Some tokens are frequent, some have no gradient."""
    g = gen(27)
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    ids = ((vocab + 1.0) ** u - 1.0).floor().clamp(0, vocab - 1).to(torch.int64 if n % 2 else torch.int32)
    ids[::5] = vocab - 1
    ids[1::97] = -1
    dy = torch.randint(-3, 4, (n, dim), device="cuda", generator=g).float()
    table = R.wrap(torch.zeros(vocab, dim, device="cuda"))
    got = ft.grad(F.embedding(table, R.wrap(ids), padding_idx=2), table, seed=R.wrap(dy)).torch()
    ref, _ = R.embedding_grad(ids, dy, vocab, 1.0, 2)
    assert torch.equal(got.double(), ref)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("padding", [-1, -2 ** 40, 8, 2 ** 32 + 5, 2 ** 33 + 5])
def test_a_padding_index_outside_the_table_is_none(index, padding):
    """Straight through the C entry point: the public function refuses it."""
    ids = torch.tensor([5, 5, 1, 5], device="cuda", dtype=index)
    dy, out = torch.ones(4, 4, device="cuda"), torch.full((8, 4), -1.0, device="cuda")
    desc = (3, 1 if index is torch.int32 else 2, 8, 4, 4, 1.0, padding)
    ws = torch.empty(_native.embedding_grad_workspace(*desc), device="cuda", dtype=torch.uint8)
    _fgt.check(_native.embedding_grad(*desc, ids.data_ptr(), dy.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(),
                                      torch.cuda.current_stream().cuda_stream))
    want = torch.zeros(8, 4, device="cuda")
    want[5], want[1] = 3.0, 1.0
    assert torch.equal(out, want)
