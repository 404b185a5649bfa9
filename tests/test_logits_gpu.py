"""Penalties, biases, grammar masks and token counts on the GPU against 64-bit oracles.

The adjusted logits are fp32 sums of a handful of terms: the tests allow 2^-21 of the terms' magnitudes (four
roundings of 2^-24, twice over), and for bf16 logits the rounding of the result (2^-9 of it, allowed twice)."""
import math

import pytest
import torch

import paged_oracle as O

pytestmark = pytest.mark.gpu
dev = "cuda"


def L():
    from lora_kernel_b200.ops import logits
    return logits


def _status_code():
    from lora_kernel_b200._ext import KernelStatusError, check_status
    try:
        check_status()
    except KernelStatusError as e:
        return str(e)
    return ""


def _table(rows, vocab, seed):
    """A counts table with every kind of entry."""
    g = torch.Generator(device=dev).manual_seed(seed)
    made = torch.randint(0, 40, (rows, vocab), device=dev, generator=g) - 30
    c = made.clamp(min=0)
    c[:, 5 % vocab] = 32767
    c -= 32768 * (torch.rand(rows, vocab, device=dev, generator=g) < 0.2).long()
    return c.to(torch.int16)


def _bits(allowed):
    """bool [m, V] -> int32 [m, ceil(V / 32)]."""
    m, v = allowed.shape
    words = (v + 31) // 32
    full = torch.zeros(m, words * 32, dtype=torch.int64, device=dev)
    full[:, :v] = allowed
    w = (full.view(m, words, 32) << torch.arange(32, device=dev)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def _compare(out, z, counts, rows, pen, biases, allowed, mask_rows):
    for i in range(z.shape[0]):
        r = None if counts is None else (i if rows is None else rows[i])
        c = counts[r].long() if r is not None and r >= 0 else None
        m = None if allowed is None else (i if mask_rows is None else mask_rows[i])
        p = tuple(pen[i].double().tolist()) if pen is not None else None
        want = O.adjust(z[i].double(), c, p, biases[i], allowed[m] if m is not None and m >= 0 else None)
        size = z[i].double().abs() * (max(p[0], 1 / p[0]) if p else 1.0)
        if c is not None:
            size = size + abs(p[1]) * (c & 0x7FFF) + abs(p[2])
        for k, b in (biases[i] or {}).items():
            size[k] += abs(b)
        got = out[i].double()
        hidden = torch.isinf(want) & (want < 0)
        assert torch.equal(torch.isneginf(got), hidden), f"row {i}: masked tokens"
        tol = 2.0 ** -21 * size + (2.0 ** -8 * want.abs() if z.dtype == torch.bfloat16 else 0.0)
        assert ((got - want).abs() <= tol)[~hidden].all(), f"row {i}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,vocab", [(1, 1), (3, 31), (2, 32), (5, 1000), (4, 2048), (3, 2049), (2, 32003), (7, 8191)])
def test_adjust_logits(dtype, n, vocab):
    ops = L()
    g = torch.Generator(device=dev).manual_seed(vocab)
    z = (torch.randn(n, vocab, device=dev, generator=g) * 4).to(dtype)
    counts = _table(n + 2, vocab, 1)
    rows = list(range(n + 2))[::-1][:n]
    if n > 2:
        rows[1] = -1
    pen = torch.stack([torch.rand(n, device=dev, generator=g) + 0.5, torch.rand(n, device=dev, generator=g) - 0.3,
                       torch.rand(n, device=dev, generator=g) * 2 - 1], dim=1)
    pen[0, 0] = 1.0
    biases = [{(7 * k + i) % vocab: (k - 3) * 1.37 for k in range(min(vocab, 40 * i))} for i in range(n)]
    allowed = torch.rand(n + 1, vocab, device=dev, generator=g) < 0.6
    allowed[n] = False  # a grammar that allows nothing
    mask_rows = [(i + 1) % (n + 1) for i in range(n)]
    mask_rows[n // 2] = -1
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    bits = _bits(allowed)
    for use in range(16):
        kw = {}
        if use & 1:
            kw.update(counts=counts, rows=t(rows), penalties=pen)
        if use & 2:
            kw.update(bias=ops.logit_bias(biases, dev))
        if use & 4:
            kw.update(mask=bits, mask_rows=t(mask_rows))
        target = z.clone()
        if use & 8:
            kw["out"] = target  # in place
        out = ops.adjust_logits(target, **kw)
        _compare(out, z, counts if use & 1 else None, rows, pen if use & 1 else None, biases if use & 2 else [None] * n,
                 allowed if use & 4 else None, mask_rows)
        assert use & 8 or torch.equal(target, z)
    assert _status_code() == ""


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,vocab", [(40, 32003), (40, 32008), (150, 6000), (150, 6001)])
def test_adjust_logits_of_many_rows(dtype, n, vocab):
    """Batches whose threads take two groups of columns, rows on and off 16 bytes; a row's last span ends inside the first
    group (6000) and inside the second (32003)."""
    ops = L()
    g = torch.Generator(device=dev).manual_seed(vocab)
    z = (torch.randn(n, vocab, device=dev, generator=g) * 4).to(dtype)
    counts = _table(n + 2, vocab, 1)
    rows = [(7 * i + 3) % (n + 2) if i % 5 else -1 for i in range(n)]
    pen = torch.rand(n, 3, device=dev, generator=g) + torch.tensor([0.5, -0.3, -0.5], device=dev)
    # columns 0, 2047, 2048 and the last one among them
    biases = [{t % vocab: (k - 3) * 1.37 for k, t in enumerate((0, 2047, 2048, 4095, 4096, vocab - 1, 97 * i, 131 * i + 5))} if i % 3 else None
              for i in range(n)]
    allowed = torch.rand(n, vocab, device=dev, generator=g) < 0.6
    mask_rows = [(i + 1) % n if i % 4 else -1 for i in range(n)]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for use in (1, 2, 4, 7, 15):
        kw = {}
        if use & 1:
            kw.update(counts=counts, rows=t(rows), penalties=pen)
        if use & 2:
            kw.update(bias=ops.logit_bias(biases, dev))
        if use & 4:
            kw.update(mask=_bits(allowed), mask_rows=t(mask_rows))
        target = z.clone()
        if use & 8:
            kw["out"] = target  # in place
        out = ops.adjust_logits(target, **kw)
        _compare(out, z, counts if use & 1 else None, rows, pen if use & 1 else None, biases if use & 2 else [None] * n,
                 allowed if use & 4 else None, mask_rows)
        assert use & 8 or torch.equal(target, z)
    assert _status_code() == ""


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_adjust_strides_and_identity_rows(dtype):
    """Row pitches of every alignment (logits, counts, masks, output), rows and mask rows left out."""
    ops = L()
    n, vocab = 4, 5003
    g = torch.Generator(device=dev).manual_seed(0)
    for pad in (0, 1, 5, 13):
        z = torch.randn(n, vocab + pad, device=dev, generator=g).to(dtype)[:, pad // 2:pad // 2 + vocab]
        counts = torch.zeros(n, vocab + pad, dtype=torch.int16, device=dev)[:, pad - pad // 2:pad - pad // 2 + vocab]
        counts.copy_(_table(n, vocab, 2))
        pen = torch.tensor([[1.3, 0.2, 0.1]] * n, device=dev)
        allowed = torch.rand(n, vocab, device=dev, generator=g) < 0.5
        words = (vocab + 31) // 32
        wide = torch.full((n, words + pad), -1, dtype=torch.int32, device=dev)
        mask = wide[:, pad // 2:pad // 2 + words]
        mask.copy_(_bits(allowed))
        hold = torch.full((n, vocab + 7 + pad), 42.0, dtype=dtype, device=dev)
        out = ops.adjust_logits(z, counts, None, pen, mask=mask, out=hold[:, 3:3 + vocab])
        _compare(out, z, counts, None, pen, [None] * n, allowed, None)
        assert (hold[:, :3] == 42).all() and (hold[:, 3 + vocab:] == 42).all()


def test_adjust_special_values():
    """Infinities and NaN in the logits: kept where allowed, -inf where not; -inf survives every penalty."""
    ops = L()
    z = torch.tensor([[math.nan, math.inf, -math.inf, 0.0, -0.0, 1.0, math.nan, math.inf, -3.0e38, 5.0]], device=dev)
    counts = torch.tensor([[1, 1, 1, 1, 1, 0, 1, 1, 1, -32768]], dtype=torch.int16, device=dev)
    pen = torch.tensor([[2.0, 0.5, 0.25]], device=dev)
    allowed = torch.tensor([[True] * 6 + [False] * 2 + [True] * 2], device=dev)
    out = ops.adjust_logits(z, counts, None, pen, mask=_bits(allowed))[0].tolist()
    assert math.isnan(out[0]) and out[1] == math.inf and out[2] == -math.inf
    assert out[3:6] == [-0.75, -0.75, 1.0] and out[6:9] == [-math.inf] * 3 and out[9] == 2.5


def test_adjust_in_place_keeps_the_rest_to_the_bit():
    """Tokens that nothing applies to keep their bits, NaN payloads among them, in place and out of place."""
    ops = L()
    n, vocab = 3, 9001
    raw = torch.randint(-2 ** 15, 2 ** 15, (n, vocab), device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(torch.int16)
    raw[(raw & 0x7F80) == 0x7F80] = 0x3F80  # finite
    z = raw.view(torch.bfloat16)
    counts = torch.zeros(n, vocab, dtype=torch.int16, device=dev)
    counts[:, 777] = 2
    pen = torch.tensor([[1.1, 0.1, 0.1]] * n, device=dev)
    bias = ops.logit_bias([{4000: 1.5}, None, {0: -1.0}], dev)
    for out in (None, z):
        got = ops.adjust_logits(z.clone() if out is None else z, counts, None, pen, bias=bias, out=out)
        same = torch.ones(n, vocab, dtype=torch.bool, device=dev)
        same[:, 777], same[0, 4000], same[2, 0] = False, False, False
        assert torch.equal(got.view(torch.int16)[same], raw[same])


@pytest.mark.parametrize("n,vocab", [(1, 3000), (40, 32003)])
def test_bias_ids_named_several_times(n, vocab):
    """Their biases add up in fp32 in the order of the list, the same in every call; other columns get their own."""
    ops = L()
    g = torch.Generator().manual_seed(5)
    for many in (2, 3, 600, 1500):
        ids = torch.cat([torch.full((many,), 77), torch.tensor([vocab - 1, 300, 77 + 256, vocab - 1])]).repeat(n)
        vals = torch.randn(n, many + 4, generator=g) * 10.0 ** torch.randint(-3, 6, (n, many + 4), generator=g)
        want = torch.zeros(n, vocab)
        for i in range(n):
            for j in range(many):
                want[i, 77] += vals[i, j]
            want[i, 300], want[i, 333] = vals[i, many + 1], vals[i, many + 2]
            want[i, vocab - 1] = vals[i, many] + vals[i, many + 3]
        bias = ((torch.arange(n + 1) * (many + 4)).to(torch.int32).to(dev), ids.to(torch.int32).to(dev), vals.reshape(-1).to(dev))
        for _ in range(3):
            got = ops.adjust_logits(torch.zeros(n, vocab, device=dev), bias=bias)
            assert torch.equal(got.cpu(), want)
    assert _status_code() == ""


def test_bad_indices_are_reported():
    ops = L()
    z = torch.randn(2, 100, device=dev)
    counts = _table(2, 100, 3)
    pen = torch.tensor([[1.5, 0.1, 0.1]] * 2, device=dev)
    t = lambda x, dt=torch.int32: torch.tensor(x, dtype=dt, device=dev)  # noqa: E731
    out = ops.adjust_logits(z, counts, t([1, 2]), pen)
    assert "out of range" in _status_code() and torch.equal(out[1], z[1]) and not torch.equal(out[0], z[0])
    bias = (t([0, 2, 3]), t([100, 4, -1]), t([1.0, 2.0, 3.0], torch.float32))
    out = ops.adjust_logits(z, bias=bias)
    assert "out of range" in _status_code()
    z2 = z.clone()
    z2[0, 4] += 2.0
    assert torch.equal(out, z2)
    out = ops.adjust_logits(z, mask=torch.zeros(1, 4, dtype=torch.int32, device=dev), mask_rows=t([0, 1]))
    assert "out of range" in _status_code() and torch.isneginf(out[0]).all() and torch.equal(out[1], z[1])
    ops.add_token_counts(counts, t([0, 5]), t([100, 3], torch.int64))
    assert "out of range" in _status_code()
    before = counts.clone()
    ops.set_token_counts(counts, t([2, -1]), t([1, 2, 3], torch.int64), t([0, 2, 3]), t([1, 1]))
    assert "out of range" in _status_code() and torch.equal(counts, before)
    ops.set_token_counts(counts, t([1]), t([1, -7, 100, 99], torch.int64), t([0, 4]), t([1]))
    assert "out of range" in _status_code()
    assert torch.equal(counts[1].long(), O.token_counts([1], [99], 100).to(dev))
    ops.set_token_counts(counts, t([1]), t([1, 2], torch.int64), t([-3, 50]), t([9]))  # offsets outside the tokens
    assert torch.equal(counts[1].long(), O.token_counts([1, 2], [], 100).to(dev))


@pytest.mark.parametrize("vocab", [1, 33, 8192, 8193, 32003, 128256])
def test_token_counts(vocab):
    ops = L()
    g = torch.Generator().manual_seed(vocab)
    histories, prompts = [], []
    for n in (0, 1, 7, 3000):
        histories.append((torch.rand(n, generator=g).pow(4) * vocab).long().clamp(max=vocab - 1).tolist())
        prompts.append(n * 2 // 3 if n != 7 else 7)
    rows = [4, 0, 5, 2]
    counts = _table(6, vocab, 4)
    before = counts.clone()
    t = lambda x, dt=torch.int32: torch.tensor(x, dtype=dt, device=dev)  # noqa: E731
    offsets = [0]
    for h in histories:
        offsets.append(offsets[-1] + len(h))
    ops.set_token_counts(counts, t(rows), t([x for h in histories for x in h], torch.int64), t(offsets), t(prompts))
    want = before.long()
    for r, h, p in zip(rows, histories, prompts):
        want[r] = O.token_counts(h[:p], h[p:], vocab).to(dev)
    assert torch.equal(counts.long(), want)
    # one more token each, the same one twice in a row of its own, and a skipped row
    toks = [vocab - 1, vocab // 2, 0, 0, vocab - 1]
    ops.add_token_counts(counts, t([4, 0, 5, 5, -1]), t(toks, torch.int64))
    for r, x in zip([4, 0, 5, 5], toks):
        want[r, x] += 1
    assert torch.equal(counts.long(), want)
    assert _status_code() == ""


def test_counts_saturate():
    ops = L()
    counts = torch.tensor([[32766, -2, 0, 32767, -1]], dtype=torch.int16, device=dev)
    for _ in range(3):
        for tok in range(5):
            ops.add_token_counts(counts, None, torch.tensor([tok], device=dev))
    assert counts[0].tolist() == [32767, -1, 3, 32767, -1]
    tokens = torch.zeros(40000, dtype=torch.int64, device=dev)
    wide = torch.zeros(1, 3, dtype=torch.int16, device=dev)
    ops.set_token_counts(wide, None, tokens, torch.tensor([0, 40000], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev))
    assert wide[0].tolist() == [32767, 0, 0]
    many = torch.zeros(1, 3, dtype=torch.int16, device=dev)
    ops.add_token_counts(many, torch.zeros(1000, dtype=torch.int32, device=dev), torch.arange(1000, device=dev) % 3)
    assert many[0].tolist() == [334, 333, 333]


def test_refusals():
    ops = L()
    z = torch.zeros(2, 64, device=dev)
    counts = torch.zeros(3, 64, dtype=torch.int16, device=dev)
    pen = torch.ones(2, 3, device=dev)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    bad = [dict(logits=z.half()), dict(logits=z.t()), dict(logits=z.cpu()), dict(counts=counts.int()), dict(counts=counts[:, :63]),
           dict(penalties=None), dict(penalties=pen[:1]), dict(penalties=pen.double()), dict(rows=i32(3)), dict(rows=i32(2).long()),
           dict(counts=counts[:1]), dict(bias=(i32(2), i32(1), pen[0, :1])), dict(bias=(i32(3), i32(1), pen[0])), dict(mask=i32(2, 1)),
           dict(mask=i32(1, 2)), dict(mask=i32(2, 2), mask_rows=i32(1)), dict(out=z[:1]), dict(out=z.bfloat16()), dict(counts=counts.cpu())]
    for kw in bad:
        a = {**dict(logits=z, counts=counts, rows=None, penalties=pen), **kw}
        with pytest.raises(RuntimeError):
            ops.adjust_logits(a.pop("logits"), a.pop("counts"), a.pop("rows"), a.pop("penalties"), **a)
    with pytest.raises(RuntimeError):
        ops.set_token_counts(counts, None, i32(4), i32(2), i32(1))
    with pytest.raises(RuntimeError):
        ops.set_token_counts(counts, None, i32(4).long(), i32(1), i32(1))
    with pytest.raises(RuntimeError):
        ops.add_token_counts(counts, i32(1), i32(2).long())
    assert ops.logit_bias([None, {}], dev) is None
    assert ops.adjust_logits(z[:0], counts, None, pen[:0]).shape == (0, 64)
