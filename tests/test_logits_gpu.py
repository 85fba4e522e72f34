"""scratchtape_b200/logits.py against a plain statement in 64 bits.

Bounds: five f32 operations (2^-24 each of the largest intermediate, below 2^-21 of |x| + frequency n + presence +
|bias|) and the result's rounding to its own type (f16 2^-11, bf16 2^-8 of it)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROUND = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}
DEV = "cuda"


def adjust(*a, **k):
    from scratchtape_b200 import logits
    return logits.adjust(*a, **k)


def want64(x, hist, prompt, rep, pres, freq, bias, masks, rows_of):
    """-> (result, the size of what was summed) in float64."""
    x = x.double().cpu().clone()
    size = x.abs().nan_to_num(0.0, posinf=0.0)
    rows, vocab = x.shape
    for r in range(rows):
        told = [t for t in hist[r]] if hist else []
        for v in set(t for t in told if 0 <= t < vocab):
            p = float(rep[r]) if rep is not None else 1.0
            x[r, v] = x[r, v] / p if x[r, v] > 0 else x[r, v] * p
            n = sum(t == v for t in told[prompt[r]:])
            f, c = (float(t[r]) if t is not None else 0.0 for t in (freq, pres))
            size[r, v] = size[r, v] * max(p, 1 / p) + abs(f) * n + abs(c)
            if n:
                x[r, v] -= f * n + c
        for v, b in (bias[r] if bias else []):
            if 0 <= v < vocab:
                x[r, v] += b
                size[r, v] += abs(b)
        m = rows_of[r] if rows_of is not None else (r if masks is not None else -1)
        if masks is not None and m >= 0:
            off = torch.tensor([not (int(masks[m, v // 32]) >> (v % 32)) & 1 for v in range(vocab)])
            x[r, off] = -math.inf
    return x, size


def ragged(lists, dtype=torch.int32):
    at = torch.tensor([0] + torch.tensor([len(x) for x in lists]).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    return torch.tensor([v for x in lists for v in x], dtype=dtype, device=DEV), at


CASES = [(1, 1, F32, 0), (3, 31, F32, 1), (4, 256, F32, 3), (2, 33, BF16, 2), (5, 1000, F16, 5), (3, 8193, BF16, 40),
         (2, 20011, F32, 300), (2, 16384, F16, 0), (1, 32768 + 9, BF16, 4000)]


@pytest.mark.parametrize("rows,vocab,dtype,length", CASES)
@pytest.mark.parametrize("inplace", [False, True])
def test_adjust(dev, rows, vocab, dtype, length, inplace):
    g = torch.Generator().manual_seed(rows * vocab + length)
    pad = 5 if inplace else 0
    wide = (torch.randn((rows, vocab + pad), generator=g) * 4).to(dtype).to(DEV)
    x = wide[:, :vocab]
    x[0, 0] = -math.inf
    draw = lambda n: [int(v) for v in (torch.rand(n, generator=g) ** 3 * vocab).long()]  # noqa: E731
    hist = [draw(length * (r + 1) // rows) + [-1, vocab, 0][:length] for r in range(rows)]
    prompt = [len(h) * (r % 3) // 3 for r, h in enumerate(hist)]
    rep, pres, freq = (torch.rand(rows, generator=g) * a + b for a, b in ((1.0, 0.8), (2.0, -1.0), (0.5, 0.0)))
    bias = [[(v, float(torch.randn((), generator=g).float())) for v in draw(r * 7 % 50)] * 2 + [(-1, 1.0), (vocab, 1.0)]
            for r in range(rows)]
    masks = torch.randint(-2 ** 31, 2 ** 31, (rows + 1, (vocab + 31) // 32), generator=g).to(torch.int32)
    masks[rows] = 0
    rows_of = [r if r % 4 else rows - r for r in range(rows)] if rows > 1 else [-1]
    for with_bias, with_mask in ((True, "rows"), (False, "own"), (True, None)):
        use = rows_of if with_mask == "rows" else None
        m = masks if with_mask else None
        want, size = want64(x, hist, prompt, rep, pres, freq, bias if with_bias else None, m, use)
        tok, at = ragged(hist)
        ids, bat = ragged([[v for v, _ in b] for b in bias])
        vals, _ = ragged([[v for _, v in b] for b in bias], F32)
        src = wide.clone()[:, :vocab] if inplace else x
        got = adjust(src, tok, at, torch.tensor(prompt, dtype=torch.int32, device=DEV), rep.to(DEV), pres.to(DEV),
                     freq.to(DEV), bias=(ids, vals, bat) if with_bias else None,
                     mask=(m.to(DEV), torch.tensor(use, dtype=torch.int32, device=DEV) if use else None)
                     if with_mask else None, out=src if inplace else None)
        dev.sync()
        if inplace:
            assert got.data_ptr() == src.data_ptr()
            assert torch.equal(src.as_strided((rows, pad), (vocab + pad, 1), vocab), wide[:, vocab:])
        got = got.double().cpu()
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine], want[~fine])
        bound = (ROUND[dtype] + 2.0 ** -21) * want.abs() + 2.0 ** -21 * size + 2.0 ** -25
        assert ((got - want)[fine].abs() <= bound[fine]).all()


def test_nothing_to_do_copies(dev):
    x = torch.randn((3, 777), device=DEV).to(BF16)
    assert torch.equal(adjust(x), x)
    assert adjust(x[:0]).shape == (0, 777)
    assert torch.equal(adjust(x.t().contiguous().t()), x)


def test_non_finite_and_masked(dev):
    x = torch.tensor([[math.nan, math.inf, -math.inf, 3.0e38, 1.0]], device=DEV)
    mask = torch.tensor([[0b11110]], dtype=torch.int32, device=DEV)
    got = adjust(x, torch.tensor([0, 1, 2, 4], dtype=torch.int32, device=DEV),
                 torch.tensor([0, 4], dtype=torch.int32, device=DEV), repetition=torch.full((1,), 2.0, device=DEV),
                 mask=(mask, None))
    want = torch.tensor([[-math.inf, math.inf, -math.inf, 3.0e38, 0.5]], device=DEV)
    assert torch.equal(got, want)
    none = adjust(x, mask=(torch.zeros_like(mask), None))
    assert (none == -math.inf).all()


def test_a_count_past_65535(dev):
    n = 70001
    x = torch.zeros((1, 40), device=DEV)
    tok = torch.full((n,), 7, dtype=torch.int32, device=DEV)
    got = adjust(x, tok, torch.tensor([0, n], dtype=torch.int32, device=DEV),
                 frequency=torch.full((1,), 0.5, device=DEV))
    assert got[0, 7] == -0.5 * n and got.abs().sum() == 0.5 * n


def test_refusals(dev):
    import scratchtape_b200._native as N
    x = torch.randn((2, 40), device=DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for bad in (lambda: adjust(x.double()), lambda: adjust(x[0]), lambda: adjust(x.cpu()),
                lambda: adjust(x, i32(1, 2)), lambda: adjust(x, i32(1, 2), i32(0, 2)),
                lambda: adjust(x, i32(1, 2).long(), i32(0, 1, 2)),
                lambda: adjust(x, repetition=torch.ones(3, device=DEV)),
                lambda: adjust(x, mask=(i32(1, 2).view(2, 1), None)),
                lambda: adjust(x, mask=(i32(1, 2, 3, 4).view(2, 2), i32(0))),
                lambda: adjust(x, bias=(i32(1), torch.ones(2, device=DEV), i32(0, 1, 1))),
                lambda: adjust(x, out=torch.empty((2, 41), device=DEV))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(N.StError, match="masks"):
        adjust(x, mask=(i32(1, 2).view(1, 2), None))
    adjust(x, mask=(i32(1, 2).view(1, 2), i32(0, 5)))
    with pytest.raises(N.StError, match="INVALID_ARG"):
        dev.sync()
    dev.sync()
