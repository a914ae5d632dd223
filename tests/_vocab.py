"""64-bit references of the vocabulary operators, written from their formulas, with the
error bounds that f32 arithmetic and one rounding to the output's type allow."""
import math

import torch

import fugatensor_b200 as ft

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32, "i64": torch.int64}
FT = {"f32": ft.fp32, "f16": ft.fp16, "bf16": ft.bf16, "i32": ft.int32, "i64": ft.int64}
U32 = 2.0 ** -24
UNIT = {"f32": U32, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # unit roundoff of the output's type
TINY = {"f32": 2.0 ** -140, "f16": 2.0 ** -25, "bf16": 2.0 ** -130}  # half the smallest subnormal step (f16), underflow (others)
# Relative error of a row's sum of exponentials: the kernels add at most 400 terms in series per
# accumulator (then trees), each term is exp of an f32 difference: |d| * e^-|d| * 2 + 4 < 5 units.
SUM_UNITS = 512 * U32


def wrap(x):
    return ft.tensor(x, dtype={v: k for k, v in zip(FT.values(), TORCH.values())}[x.dtype])


def check(got, ref, bound, what=""):
    """got within bound of ref elementwise; NaN and infinities in the same places."""
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(inf, torch.isinf(got)) and torch.equal(got[inf], ref[inf]), f"{what}: infinities in other places"
    ok = torch.isfinite(ref)
    err, bound = (got - ref).abs()[ok], bound.expand_as(ref)[ok]
    if err.numel():
        worst = int((err - bound).argmax())
        assert bool((err <= bound).all()), f"{what}: error {err[worst]:.3g} over {bound[worst]:.3g} at {ref[ok][worst]:.6g}"


def rounded(bound32, ref, dtype):
    """bound32 (error before the final rounding) plus that rounding."""
    size = ref.double().abs().nan_to_num(posinf=0.0)
    return bound32 + UNIT[dtype] * (size + bound32) + TINY[dtype]


def embedding(table, ids, scale):
    inside = (ids >= 0) & (ids < table.shape[0])
    rows = table.double()[torch.where(inside, ids, 0).long()] if table.shape[0] else torch.zeros(
        *ids.shape, table.shape[1], dtype=torch.float64, device=table.device)
    return torch.where(inside[..., None], rows * scale, 0.0)


def embedding_grad(ids, dy, vocab, scale, padding):
    """(gradient, sum of |dy| times the number of terms) per element."""
    ids, dy = ids.reshape(-1), dy.reshape(ids.numel(), -1).double()
    keep = (ids >= 0) & (ids < vocab)
    if padding is not None:
        keep &= ids != padding
    out = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device=dy.device)
    size = torch.zeros_like(out)
    out.index_add_(0, ids[keep].long(), dy[keep])
    size.index_add_(0, ids[keep].long(), dy[keep].abs())
    terms = torch.bincount(ids[keep].long(), minlength=vocab)[:, None]
    return out * scale, size * abs(scale) * (terms + 2)


def cross_entropy(x, t, ignore=-100, eps=0.0, z=0.0, reduction="mean", seed=None):
    """(loss, its bound, gradient, its bound before rounding) of x [rows, vocab]."""
    x, v = x.double(), x.shape[-1]
    counted = (t != ignore) & (t >= 0) & (t < v)
    at = torch.where(counted, t, 0).long()
    lse = torch.logsumexp(x, 1)
    lse = torch.where((x == -math.inf).all(1), math.nan, lse)
    xt = x.gather(1, at[:, None])[:, 0]
    row = lse - (1.0 - eps) * xt
    size = 1.0 + lse.abs() + xt.abs().nan_to_num(posinf=0.0)
    if eps:
        row = row - eps / v * x.sum(1)
        size = size + eps / v * x.abs().sum(1).nan_to_num(posinf=0.0)
    if z:
        row = row + z * lse ** 2
        size = size + 3.0 * z * (lse ** 2 + lse.abs())
    row, size = torch.where(counted, row, 0.0), torch.where(counted, size, 0.0)
    p = torch.exp(x - lse[:, None])
    hit = torch.zeros_like(x)
    hit.scatter_(1, at[:, None], 1.0)
    d = p * (1.0 + 2.0 * z * lse[:, None]) - (1.0 - eps) * hit - eps / v
    dsize = p * (3.0 * SUM_UNITS * (1.0 + 2.0 * z * lse[:, None].abs()) + 8.0 * z * U32 * lse[:, None].abs()) + 8.0 * U32 * (hit + eps / v + d.abs())
    n = max(1, int(counted.sum()))
    w = torch.ones_like(row) if seed is None else seed.double().expand_as(row)
    g = w / n if reduction == "mean" else w
    d, dsize = (torch.where(counted[:, None], q * k[:, None], 0.0) for q, k in ((d, g), (dsize, g.abs())))
    if reduction == "none":
        return row, SUM_UNITS * size, d, dsize
    total, bound = row.sum(), SUM_UNITS * size.sum()
    return (total / n, bound / n, d, dsize) if reduction == "mean" else (total, bound, d, dsize)


def adjust_logits(x, tokens=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0,
                  bias_tokens=None, bias=None, allowed=None):
    """(result, bound before rounding) of x [rows, vocab]; a loop over rows."""
    rows, v = x.shape
    out, size = x.double().clone(), x.double().abs().nan_to_num(0.0, 0.0, 0.0)

    def of(p, i):
        return float(p[i]) if isinstance(p, torch.Tensor) else p

    for i in range(rows):
        if tokens is not None:
            n = min(max(int(lengths[i]), 0), tokens.shape[1]) if lengths is not None else tokens.shape[1]
            p = min(max(int(prompt_lengths[i]), 0), n) if prompt_lengths is not None else 0
            line = tokens[i, :n].long()
            inside = (line >= 0) & (line < v)
            seen = torch.bincount(line[inside], minlength=v)
            made = torch.bincount(line[p:][inside[p:]], minlength=v)
            r, f, a = of(repetition, i), of(frequency, i), of(presence, i)
            out[i] = torch.where(seen > 0, torch.where(out[i] > 0, out[i] / r, out[i] * r), out[i])
            out[i] -= f * made + a * (made > 0)
            size[i] = size[i] * max(r, 1.0 / r) + abs(f) * made + abs(a)
        if bias is not None:
            ids = bias_tokens[i].long()
            inside = (ids >= 0) & (ids < v)
            out[i].index_add_(0, ids[inside], bias[i][inside].double())
            size[i].index_add_(0, ids[inside], bias[i][inside].double().abs() * ids.numel())
        if allowed is not None:
            bits = torch.arange(v, device=x.device)
            out[i][(allowed[i].long()[bits // 32] >> (bits % 32)) & 1 == 0] = -math.inf
    return out, 8.0 * U32 * size
