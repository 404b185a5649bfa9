"""The page-scaled 8-bit KV cache on the GPU against 64-bit oracles.

Appending and reading back are exact: scales are powers of two, so every step is a product with a power of two and
one rounding that the oracle repeats.  Attention rounds the softmax weights to 11 bits (2^-11 of sum p|v|; the scores
and the sums are fp32) and its result to bf16 (2^-9 of it); the tests allow twice that."""
import math

import pytest
import torch

import paged_oracle as O

pytestmark = pytest.mark.gpu
dev = "cuda"
KINDS = ["fp8_page", "int8_page"]


def P():
    from lora_kernel_b200.ops import paged
    return paged


def _status_code():
    from lora_kernel_b200._ext import KernelStatusError, check_status
    try:
        check_status()
    except KernelStatusError as e:
        return str(e)
    return ""


def _same(got_codes, got_scale, ref, what):
    assert torch.equal(got_scale.double(), ref.scale), what + ": scales"
    assert torch.equal(got_codes.double(), ref.codes), what + ": codes"


def _cache(kind, pages, page, Hkv, Dh):
    return [t[0] for t in P().new_page_cache(1, pages, page, Hkv, Dh, kind, dev)]


def _garbage(cache, seed):
    """Any bytes in the codes (NaN among the e4m3 ones), NaN in the scales."""
    k, v, ks, vs = cache
    g = torch.Generator(device=dev).manual_seed(seed)
    for c in (k, v):
        c.view(torch.uint8).copy_(torch.randint(0, 256, c.shape, device=dev, generator=g, dtype=torch.int32).to(torch.uint8))
    ks.fill_(math.nan)
    vs.fill_(math.nan)


def _slots(table, page, a, b):
    return [table[t // page] * page + t % page for t in range(a, b)]


# ------------------------------------------------------------------ append, read-back
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,Hkv,Dh,page", [(4, 2, 64, 16), (8, 1, 128, 7), (3, 3, 64, 1), (16, 8, 128, 40), (0, 5, 64, 24)])
def test_append_in_pieces(kind, Hq, Hkv, Dh, page):
    paged = P()
    g = torch.Generator(device=dev).manual_seed(1)
    pages = 40
    k, v, ks, vs = cache = _cache(kind, pages, page, Hkv, Dh)
    _garbage(cache, 2)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).tolist()
    lens = [0, 0, 0]
    tables = [order[i * 12:(i + 1) * 12] for i in range(3)]
    refk, refv = O.PageCache(k, ks, page), O.PageCache(v, vs, page)
    touched = set()
    for step, takes in enumerate([(1, 1, 3), (1, 5, 0), (1, 1, 1), (2 * page, 1, page), (3, page + 1, 2)]):
        takes = [min(t, 12 * page - n) for t, n in zip(takes, lens)]
        slots = [s for i, t in enumerate(takes) for s in _slots(tables[i], page, lens[i], lens[i] + t)]
        lens = [n + t for n, t in zip(lens, takes)]
        x = torch.randn(len(slots), (Hq + 2 * Hkv) * Dh, device=dev, generator=g) * 2.0 ** (step - 1)
        wide = torch.zeros(len(slots), x.shape[1] + 24, dtype=torch.bfloat16, device=dev)  # a row pitch of its own
        qkv = wide[:, :x.shape[1]]
        qkv.copy_(x)
        paged.page_append(qkv, Hq, Hkv, Dh, torch.tensor(slots, dtype=torch.int32, device=dev), k, v, ks, vs, page)
        rows = qkv.view(len(slots), Hq + 2 * Hkv, Dh)
        refk.append(rows[:, Hq:Hq + Hkv], slots)
        refv.append(rows[:, Hq + Hkv:], slots)
        touched |= set(slots)
        at = torch.tensor(sorted(touched), device=dev)
        for got, sc, ref in ((k, ks, refk), (v, vs, refv)):
            assert torch.equal(got[at].double(), ref.codes[at]), f"step {step}: codes"
            assert torch.equal(sc[at // page].double(), ref.scale[at // page]), f"step {step}: scales"
        rest = torch.ones(pages * page, dtype=torch.bool, device=dev)
        rest[at] = False
        assert torch.equal(k[rest].double().nan_to_num(7.5), refk.codes[rest].nan_to_num(7.5)), "slots not appended to"
        out = torch.zeros(len(at), 2 * Hkv * Dh + 8, dtype=torch.bfloat16, device=dev)[:, :2 * Hkv * Dh]
        paged.page_gather(k, v, ks, vs, at.to(torch.int32), Hkv, Dh, page, out=out)
        want = torch.stack([refk.values(at), refv.values(at)], dim=1).reshape(len(at), -1)
        assert torch.equal(out.double(), want), f"step {step}: read back"
    assert _status_code() == ""


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1, 7, 16, 40, 256])
@pytest.mark.parametrize("rows", [600, 2100])
def test_append_many_rows(kind, page, rows):
    """Calls whose warps look for runs in windows of several rows: three sequences that go on inside a page (the page's
    scale grows), skipped rows between them, runs across window borders and longer than a warp looks at once."""
    paged = P()
    Hkv, Dh = 1, 64
    g = torch.Generator(device=dev).manual_seed(page)
    starts = [0, page // 2, 3 * page + page // 3]
    takes = [rows // 2, rows // 3, rows - rows // 2 - rows // 3]
    need = [-(-(s + t) // page) for s, t in zip(starts, takes)]
    pages = sum(need) + 3
    k, v, ks, vs = cache = _cache(kind, pages, page, Hkv, Dh)
    _garbage(cache, 2)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).tolist()
    tables = [[order.pop() for _ in range(n)] for n in need]
    cpu = [O.PageCache(c.cpu(), s.cpu(), page) for c, s in ((k, ks), (v, vs))]
    held = [_slots(t, page, 0, n) for t, n in zip(tables, starts)]
    new = [_slots(t, page, n, n + m) + [-1] * 3 for t, n, m in zip(tables, starts, takes)]
    for slots, size in ((sum(held, []), 1.0), (sum(new, []), 4.0)):
        x = torch.randn(len(slots), 2 * Hkv, Dh, device=dev, generator=g) * size
        x = (x * torch.exp2(torch.randint(-3, 4, (len(slots), 1, 1), device=dev, generator=g).float())).to(torch.bfloat16)
        paged.page_append(x.view(len(slots), -1), 0, Hkv, Dh, torch.tensor(slots, dtype=torch.int32, device=dev), k, v, ks, vs, page)
        cpu[0].append(x[:, :Hkv].cpu(), slots)
        cpu[1].append(x[:, Hkv:].cpu(), slots)
    at = torch.tensor(sorted(s for s in sum(held + new, []) if s >= 0))
    for got, sc, ref in ((k, ks, cpu[0]), (v, vs, cpu[1])):
        assert torch.equal(got.cpu()[at].double(), ref.codes[at])
        assert torch.equal(sc.cpu()[at // page].double(), ref.scale[at // page])
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[at] = False
    assert torch.equal(k.cpu()[rest].double().nan_to_num(7.5), cpu[0].codes[rest].nan_to_num(7.5)), "slots not appended to"
    assert _status_code() == ""


@pytest.mark.parametrize("kind", KINDS)
def test_append_edges(kind):
    """Zeros, subnormals, the largest values, infinities and NaN; skipped rows; boundaries of the scale."""
    paged = P()
    Hq, Hkv, Dh, page = 1, 2, 64, 8
    k, v, ks, vs = cache = _cache(kind, 16, page, Hkv, Dh)
    _garbage(cache, 5)
    refk, refv = O.PageCache(k, ks, page), O.PageCache(v, vs, page)
    q = O.QMAX[k.dtype]
    rows = torch.zeros(12, 5, Dh, device=dev)
    rows[1] = 1e-39
    rows[2] = 3.3e38
    rows[3, :, ::2], rows[3, :, 1::2] = math.inf, 1.0
    rows[4, :, ::3], rows[4, :, 1::3] = math.nan, -2.0
    rows[5], rows[5, :, 0] = math.nan, -math.inf
    rows[6] = q            # exactly QMAX * 2^0
    rows[7] = q * 1.0078125  # the next bf16 above it (where it has one)
    rows[8] = -q * 2.0 ** -30
    rows[9], rows[10], rows[11] = 1.0, 300.0, 2.0 ** -100
    qkv = rows.to(torch.bfloat16).view(12, -1)
    slots = [0, 8, 16, 24, 32, 40, 48, 56, 64, 72, -1, 80]
    slots_t = torch.tensor(slots, dtype=torch.int32, device=dev)
    paged.page_append(qkv, Hq, Hkv, Dh, slots_t, k, v, ks, vs, page)
    r = qkv.view(12, 5, Dh)
    refk.append(r[:, 1:3], slots)
    refv.append(r[:, 3:], slots)
    at = torch.tensor([s for s in slots if s >= 0], device=dev)
    for got, sc, ref in ((k, ks, refk), (v, vs, refv)):
        assert torch.equal(got[at].double(), ref.codes[at])
        assert torch.equal(sc[at // page].double(), ref.scale[at // page])
        assert torch.isfinite(got[at].float()).all()
    assert float(ks[0, 0]) == 2.0 ** -126 and float(ks[6, 0]) == 1.0 and float(ks[7, 0]) == 2.0


def test_append_one_by_one_is_append_at_once():
    """e4m3: raising a page's scale moves exponents only, as long as no code becomes subnormal."""
    paged = P()
    Hkv, Dh, page = 2, 128, 16
    g = torch.Generator(device=dev).manual_seed(9)
    x = (torch.rand(page, 2 * Hkv * Dh, device=dev, generator=g) + 1.0) * 2.0 ** torch.arange(page, device=dev).remainder(5)[:, None]
    qkv = x.to(torch.bfloat16)
    a, b = _cache("fp8_page", 2, page, Hkv, Dh), _cache("fp8_page", 2, page, Hkv, Dh)
    slots = torch.arange(page, dtype=torch.int32, device=dev) + page
    paged.page_append(qkv, 0, Hkv, Dh, slots, *a, page)
    for t in range(page):
        paged.page_append(qkv[t:t + 1], 0, Hkv, Dh, slots[t:t + 1], *b, page)
    for u, w in zip(a, b):
        assert torch.equal(u.float(), w.float())


def test_append_and_gather_report_bad_slots():
    paged = P()
    Hkv, Dh, page = 1, 64, 4
    k, v, ks, vs = _cache("fp8_page", 4, page, Hkv, Dh)
    qkv = torch.ones(2, 2 * Dh, dtype=torch.bfloat16, device=dev)
    paged.page_append(qkv, 0, Hkv, Dh, torch.tensor([2, 16], dtype=torch.int32, device=dev), k, v, ks, vs, page)
    assert "out of range" in _status_code()
    assert float(k[2].float().sum()) == 64 * 256.0 and float(ks[0, 0]) == 2.0 ** -8
    got = paged.page_gather(k, v, ks, vs, torch.tensor([2, 99, -1], dtype=torch.int32, device=dev), Hkv, Dh, page)
    assert "out of range" in _status_code()
    assert torch.equal(got.float(), torch.tensor([1.0, 0.0, 0.0], device=dev)[:, None].expand(3, 128))


# ------------------------------------------------------------------ attention
def _filled(kind, ctxs, page, Hkv, Dh, seed, spread=0.0):
    """A cache holding sequences of these lengths (appended whole), everything else garbage; and the oracle's values.
    spread: the values of a page are scaled by a random power of two in [-spread, spread]."""
    paged = P()
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-c // page) for c in ctxs]
    pages = sum(need) + 5
    k, v, ks, vs = cache = _cache(kind, pages, page, Hkv, Dh)
    _garbage(cache, seed + 1)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    tables = [[order.pop() for _ in range(n)] for n in need]
    width = max(1, max(need)) + 1
    bt = torch.full((len(ctxs), width), -1, dtype=torch.int32)  # entries past a sequence's pages are never read
    refs = []
    for i, c in enumerate(ctxs):
        bt[i, :need[i]] = torch.tensor(tables[i], dtype=torch.int32)
        x = torch.randn(c, 2 * Hkv, Dh, device=dev, generator=g)
        if spread:
            e = torch.randint(-int(spread), int(spread) + 1, (need[i],), device=dev, generator=g)
            x[:, Hkv:] *= torch.exp2(e.float()).repeat_interleave(page)[:c, None, None]
        qkv = x.reshape(c, 2 * Hkv * Dh).to(torch.bfloat16)
        slots = torch.tensor(_slots(tables[i], page, 0, c), dtype=torch.int32, device=dev)
        if c:
            paged.page_append(qkv, 0, Hkv, Dh, slots, k, v, ks, vs, page)
            both = paged.page_gather(k, v, ks, vs, slots, Hkv, Dh, page).double().view(c, 2, Hkv, Dh)
            refs.append((both[:, 0], both[:, 1]))
        else:
            refs.append((x[:, :Hkv].double(), x[:, Hkv:].double()))
    return cache, bt.to(dev), refs


def _check_attention(out, q, refs, ctxs, q_len, Hq, Dh, scale=None):
    q = q.double().view(len(ctxs), q_len, Hq, Dh)
    out = out.double().view(len(ctxs), q_len, Hq, Dh)
    for i, c in enumerate(ctxs):
        want, mag = O.attention(q[i], *refs[i], c, q_len, scale)
        err = (out[i] - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * mag).all(), f"seq {i} (ctx {c}): worst {float(err.max()):.3g}"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,Hkv,Dh,page,q_len", [
    (4, 2, 64, 16, 1), (8, 1, 128, 16, 1), (32, 8, 128, 16, 1), (3, 3, 64, 7, 1), (7, 1, 128, 24, 1), (16, 1, 64, 32, 1),
    (24, 8, 128, 1, 1), (4, 1, 128, 16, 5), (16, 4, 64, 24, 3), (8, 8, 64, 16, 17), (5, 1, 128, 256, 9), (40, 2, 64, 13, 2)])
def test_attention(kind, Hq, Hkv, Dh, page, q_len):
    ctxs = [1, 0, 2, 15, 16, 17, 33, 64, 127, 300, 1025]
    (k, v, ks, vs), bt, refs = _filled(kind, ctxs, page, Hkv, Dh, 11)
    g = torch.Generator(device=dev).manual_seed(12)
    heads = Hq + 2 * Hkv
    qkv = torch.randn(len(ctxs) * q_len, heads * Dh, device=dev, generator=g).to(torch.bfloat16)
    q = qkv[:, :Hq * Dh]
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=dev)
    for max_ctx in (0, 1025):
        out = P().page_attention(q, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh, q_len=q_len, max_ctx=max_ctx)
        _check_attention(out, q, refs, ctxs, q_len, Hq, Dh)
    assert _status_code() == ""


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,Hkv,Dh,q_len,ctxs", [(4, 1, 128, 1, [20011]), (8, 2, 64, 4, [9000, 1, 70]), (1, 1, 64, 1, [5, 30000])])
def test_attention_long(kind, Hq, Hkv, Dh, q_len, ctxs):
    """A long axis split over many blocks, beside short ones."""
    (k, v, ks, vs), bt, refs = _filled(kind, ctxs, 16, Hkv, Dh, 21)
    q = torch.randn(len(ctxs) * q_len, Hq * Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(torch.bfloat16)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=dev)
    wide = torch.zeros(q.shape[0], Hq * Dh + 8, dtype=torch.bfloat16, device=dev)
    out = P().page_attention(q, k, v, ks, vs, bt, ctx, 16, Hq, Hkv, Dh, q_len=q_len, max_ctx=max(ctxs), out=wide[:, :Hq * Dh])
    _check_attention(out, q, refs, ctxs, q_len, Hq, Dh)
    assert not wide[:, Hq * Dh:].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,Hkv,Dh,q_len,ctxs", [
    (8, 1, 128, 1, [3900]), (6, 1, 128, 3, [4100]), (2, 1, 64, 1, [5003]), (16, 2, 64, 2, [4000, 10, 0, 2500]), (12, 2, 128, 1, [1025, 1024]),
    (24, 2, 64, 5, [3000, 777])])
def test_attention_parts(kind, Hq, Hkv, Dh, q_len, ctxs):
    """Contexts cut into 2 to 16 parts, joined by their cluster, and (a longer bound) into more, joined by a second
    launch: both against the oracle; parts without a token among them."""
    (k, v, ks, vs), bt, refs = _filled(kind, ctxs, 16, Hkv, Dh, 81)
    q = torch.randn(len(ctxs) * q_len, Hq * Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(torch.bfloat16)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=dev)
    wide = torch.cat([bt, torch.full((len(ctxs), 8000), -1, dtype=torch.int32, device=dev)], dim=1)
    for table, max_ctx in ((bt, max(ctxs)), (bt, 0), (wide, 0), (wide, 1000)):
        out = P().page_attention(q, k, v, ks, vs, table, ctx, 16, Hq, Hkv, Dh, q_len=q_len, max_ctx=max_ctx)
        _check_attention(out, q, refs, ctxs, q_len, Hq, Dh)
    assert _status_code() == ""


@pytest.mark.parametrize("kind", KINDS)
def test_attention_full_batch_with_long_bounds(kind):
    """A batch that fills the GPU, two long contexts in it, with bounds from below the longest to far above it."""
    Hq, Hkv, Dh, page = 16, 8, 64, 16
    ctxs = [(37 * i) % 90 for i in range(158)] + [5000, 9001]
    (k, v, ks, vs), bt, refs = _filled(kind, ctxs, page, Hkv, Dh, 21)
    q = torch.randn(len(ctxs), Hq * Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(torch.bfloat16)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=dev)
    wide = torch.cat([bt, torch.full((len(ctxs), 8192), -1, dtype=torch.int32, device=dev)], dim=1)
    for table, max_ctx in ((bt, 9001), (bt, 90), (wide, 32768), (wide, 0)):
        out = P().page_attention(q, k, v, ks, vs, table, ctx, page, Hq, Hkv, Dh, max_ctx=max_ctx)
        _check_attention(out, q, refs, ctxs, 1, Hq, Dh)
    assert _status_code() == ""


def test_attention_full_batch_takes_no_longer_for_a_longer_bound():
    """A captured step passes the longest context that the server allows: the same work must not wait for parts without
    tokens (up to 300 tokens in a batch of 1024 blocks took nine times as long for a bound of 32768)."""
    Hq, Hkv, Dh, page, n = 32, 8, 128, 16, 128
    k, v, ks, vs = _cache("fp8_page", 1024, page, Hkv, Dh)
    ks.fill_(1.0)
    vs.fill_(1.0)
    bt = torch.randint(0, 1024, (n, 32768 // page), device=dev, dtype=torch.int32, generator=torch.Generator(device=dev).manual_seed(1))
    ctx = (torch.arange(n, device=dev) * 7 % 300 + 1).to(torch.int32)
    q = torch.randn(n, Hq * Dh, device=dev).to(torch.bfloat16)

    def us(max_ctx):
        best = 1e9
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(20):
                P().page_attention(q, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh, max_ctx=max_ctx)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) * 50)
        return best

    us(4096)
    base = us(4096)
    for bound in (4097, 8192, 32768):
        assert us(bound) < 2 * base


@pytest.mark.parametrize("kind", KINDS)
def test_attention_scales_far_apart(kind):
    """Pages whose values differ by 2^40: a query that looks at a page of small values still sees them."""
    Hq, Hkv, Dh, page, ctxs = 4, 1, 64, 8, [200, 31]
    (k, v, ks, vs), bt, refs = _filled(kind, ctxs, page, Hkv, Dh, 31, spread=20)
    for factor in (1.0, 30.0, 2.0 ** -40, 2.0 ** 20):
        # queries of every size: each along one key, so that large ones look at one page only
        q = torch.stack([refs[i][0][c * 3 // 4, 0].expand(Hq, Dh) for i, c in enumerate(ctxs)]).reshape(2, -1)
        q = (q * factor * torch.tensor([1.0, 2.0 ** -10, 8.0, -1.0], device=dev).repeat_interleave(Dh)).to(torch.bfloat16)
        ctx = torch.tensor(ctxs, dtype=torch.int32, device=dev)
        out = P().page_attention(q, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh)
        qq = q.double().view(2, 1, Hq, Dh)
        for i, c in enumerate(ctxs):
            want, mag = O.attention(qq[i], *refs[i], c, 1)
            err = (out[i].double().view(1, Hq, Dh) - want).abs()
            # large scores: fp32 keeps 2^-24 of the score in the exponent
            top = float((qq[i, 0] @ refs[i][0][:, 0].T).abs().max()) / math.sqrt(Dh) * 1.4427
            assert (err <= 2.0 ** -8 * want.abs() + (2.0 ** -10 + top * 2.0 ** -21) * mag).all(), (factor, i, float(err.max()))


def test_attention_zero_pages_and_scale_argument():
    """All-zero keys and values (scale 2^-126) beside ordinary ones; a scale of the caller's."""
    paged = P()
    Hq, Hkv, Dh, page, c = 8, 2, 64, 16, 80
    k, v, ks, vs = cache = _cache("fp8_page", 8, page, Hkv, Dh)
    _garbage(cache, 3)
    x = torch.randn(c, 2 * Hkv, Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    x[16:48] = 0.0
    x[48:64, :Hkv] = 0.0
    slots = torch.arange(c, dtype=torch.int32, device=dev)
    paged.page_append(x.reshape(c, -1).to(torch.bfloat16), 0, Hkv, Dh, slots, k, v, ks, vs, page)
    both = paged.page_gather(k, v, ks, vs, slots, Hkv, Dh, page).double().view(c, 2, Hkv, Dh)
    bt = torch.arange(5, dtype=torch.int32, device=dev).view(1, 5)
    q = torch.randn(1, Hq * Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(5)).to(torch.bfloat16)
    for ctx in (80, 48, 33):
        t = torch.tensor([ctx], dtype=torch.int32, device=dev)
        for scale in (None, 0.02, 0.0):
            out = paged.page_attention(q, k, v, ks, vs, bt, t, page, Hq, Hkv, Dh, scale=scale)
            _check_attention(out, q, [(both[:ctx, 0], both[:ctx, 1])], [ctx], 1, Hq, Dh, scale)
    only = torch.tensor([1, 2, 1, 2, 1], dtype=torch.int32, device=dev).view(1, 5)  # zero pages alone
    out = paged.page_attention(q, k, v, ks, vs, only, torch.tensor([80], dtype=torch.int32, device=dev), page, Hq, Hkv, Dh)
    assert not out.any()


def test_attention_nan_query_and_future_tokens():
    """A NaN query spoils its own row alone; tokens after a query's position do not reach it."""
    paged = P()
    Hq, Hkv, Dh, page, c, q_len = 4, 1, 64, 16, 40, 3
    (k, v, ks, vs), bt, refs = _filled("fp8_page", [c], page, Hkv, Dh, 41)
    q = torch.randn(q_len, Hq * Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(2)).to(torch.bfloat16)
    ctx = torch.tensor([c], dtype=torch.int32, device=dev)
    base = paged.page_attention(q, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh, q_len=q_len)
    q2 = q.clone()
    q2[1, :Dh] = math.nan
    out = paged.page_attention(q2, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh, q_len=q_len)
    assert torch.isnan(out[1, :Dh].float()).all()
    out[1, :Dh] = base[1, :Dh]
    assert torch.equal(out, base)
    # the last token replaced: queries 0 and 1 keep their bits
    slot = int(bt[0, (c - 1) // page]) * page + (c - 1) % page
    k[slot] = 0.5
    v[slot] = 448.0
    out = paged.page_attention(q, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh, q_len=q_len)
    assert torch.equal(out[:2], base[:2]) and not torch.equal(out[2], base[2])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,Hkv,Dh,q_len", [(4, 1, 64, 1), (4, 1, 128, 3), (8, 2, 64, 5), (1, 1, 128, 7)])
def test_attention_query_rows_far_apart(kind, Hq, Hkv, Dh, q_len):
    """Query rows (heads, tokens) 2^30 to 2^120 above their neighbours in a tile: the others keep their bits."""
    page, ctxs = 16, [70, 333]
    (k, v, ks, vs), bt, refs = _filled(kind, ctxs, page, Hkv, Dh, 91)
    g = torch.Generator(device=dev).manual_seed(92)
    q = torch.randn(2 * q_len, Hq, Dh, device=dev, generator=g).to(torch.bfloat16)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=dev)

    def call(x):
        return P().page_attention(x.view(2 * q_len, Hq * Dh), k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh, q_len=q_len).view(2 * q_len, Hq, Dh)

    base = call(q)
    _check_attention(base, q, refs, ctxs, q_len, Hq, Dh)
    big = torch.arange(2 * q_len * Hq, device=dev).view(2 * q_len, Hq) % 3 == 1
    for e in (30, 60, 120):
        out = call(torch.where(big[:, :, None], q * 2.0 ** e, q))
        assert torch.equal(out[~big], base[~big])


def test_attention_reports_bad_page_ids():
    """A page id outside the cache is recorded, its tokens are left out, nothing is read there."""
    Hq, Hkv, Dh, page = 4, 1, 64, 16
    (k, v, ks, vs), bt, refs = _filled("fp8_page", [64, 20], page, Hkv, Dh, 51)
    q = torch.randn(2, Hq * Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(2)).to(torch.bfloat16)
    ctx = torch.tensor([64, 20], dtype=torch.int32, device=dev)
    bad = bt.clone()
    bad[0, 1] = 1 << 30
    bad[1, 0], bad[1, 1] = -5, k.shape[0] // page
    out = P().page_attention(q, k, v, ks, vs, bad, ctx, page, Hq, Hkv, Dh)
    assert "out of range" in _status_code()
    keep = torch.tensor([t for t in range(64) if t // page != 1], device=dev)
    _check_attention(out[:1], q[:1], [(refs[0][0][keep], refs[0][1][keep])], [48], 1, Hq, Dh)
    assert not out[1].any()
    long = torch.tensor([64, 1 << 20], dtype=torch.int32, device=dev)  # longer than its table
    bt[1] = bt[0]
    P().page_attention(q, k, v, ks, vs, bt, long, page, Hq, Hkv, Dh)
    assert "out of range" in _status_code()


def test_offsets_past_32_bits():
    """A cache of more than 2^31 codes: its last pages are written, read, attended to and copied."""
    paged = P()
    Hq, Hkv, Dh, page = 8, 8, 128, 16
    pages = (2 ** 31 // (Hkv * Dh) + 4096) // page
    k, v, ks, vs = [t[0] for t in paged.new_page_cache(1, pages, page, Hkv, Dh, "fp8_page", dev)]
    c = 40
    table = [pages - 1, 1, pages - 2]
    slots = torch.tensor(_slots(table, page, 0, c), dtype=torch.int32, device=dev)
    qkv = torch.randn(c, (Hq + 2 * Hkv) * Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(2)).to(torch.bfloat16)
    paged.page_append(qkv, Hq, Hkv, Dh, slots, k, v, ks, vs, page)
    got = paged.page_gather(k, v, ks, vs, slots, Hkv, Dh, page)
    ref = O.PageCache(torch.zeros(3 * page, Hkv, Dh, dtype=k.dtype, device=dev), torch.zeros(3, Hkv, device=dev), page)
    rows = qkv.view(c, Hq + 2 * Hkv, Dh)
    ref.append(rows[:, Hq:Hq + Hkv], list(range(c)))
    assert torch.equal(got[:, :Hkv * Dh].double(), ref.values(torch.arange(c, device=dev)).view(c, -1))
    bt = torch.tensor([table], dtype=torch.int32, device=dev)
    ctx = torch.tensor([c], dtype=torch.int32, device=dev)
    both = got.double().view(c, 2, Hkv, Dh)
    q = qkv[:1, :Hq * Dh]
    out = paged.page_attention(q, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh)
    _check_attention(out, q, [(both[:, 0], both[:, 1])], [c], 1, Hq, Dh)
    paged.copy_pages([t[None] for t in (k, v, ks, vs)], [(pages - 1, 0), (pages - 2, pages - 3)], pages)
    bt2 = torch.tensor([[0, 1, pages - 3]], dtype=torch.int32, device=dev)
    assert torch.equal(paged.page_attention(q, k, v, ks, vs, bt2, ctx, page, Hq, Hkv, Dh), out)


def test_attention_streams_and_graphs():
    """On a stream of its own and replayed from a CUDA graph with lengths that changed since the capture."""
    Hq, Hkv, Dh, page, ctxs = 8, 2, 128, 16, [700, 20, 3000]
    (k, v, ks, vs), bt, refs = _filled("fp8_page", ctxs, page, Hkv, Dh, 61)
    q = torch.randn(3, Hq * Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(2)).to(torch.bfloat16)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=dev)

    def call():
        return P().page_attention(q, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh, max_ctx=3000)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = call()
    s.synchronize()
    _check_attention(out, q, refs, ctxs, 1, Hq, Dh)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for lens in (ctxs, [1, 0, 2999], [0, 0, 0]):
        ctx.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        _check_attention(out, q, [(a[:c], b[:c]) for (a, b), c in zip(refs, lens)], lens, 1, Hq, Dh)


def test_long_context_in_a_graph():
    """More parts than a cluster joins (a second launch that starts early), captured and replayed over changing lengths,
    with another kernel's output as its query."""
    Hq, Hkv, Dh, page, c = 4, 1, 64, 16, 20000
    (k, v, ks, vs), bt, refs = _filled("fp8_page", [c], page, Hkv, Dh, 65)
    q0 = torch.randn(1, Hq * Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(2)).to(torch.bfloat16)
    ctx = torch.tensor([c], dtype=torch.int32, device=dev)

    def call():
        q = q0 * 2
        out = P().page_attention(q, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh, max_ctx=c)
        return out + 1  # reads the result at once

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n in (c, 1, 0, 333, c - 1):
        ctx.fill_(n)
        graph.replay()
        graph.replay()
        want, mag = O.attention((q0 * 2).double().view(1, Hq, Dh), *[x[:n] for x in refs[0]], n, 1)
        err = (out.double().view(1, Hq, Dh) - 1 - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * mag + 2.0 ** -8).all()  # + 1 in bf16: 2^-8


def test_attention_repeats_to_the_bit():
    Hq, Hkv, Dh, page, ctxs = 4, 1, 128, 16, [9000, 333]
    (k, v, ks, vs), bt, _ = _filled("fp8_page", ctxs, page, Hkv, Dh, 71)
    q = torch.randn(2, Hq * Dh, device=dev, generator=torch.Generator(device=dev).manual_seed(2)).to(torch.bfloat16)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=dev)
    first = P().page_attention(q, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh, max_ctx=9000)
    for _ in range(5):
        assert torch.equal(P().page_attention(q, k, v, ks, vs, bt, ctx, page, Hq, Hkv, Dh, max_ctx=9000), first)


def test_empty_batches():
    paged = P()
    k, v, ks, vs = _cache("int8_page", 2, 16, 1, 64)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    paged.page_append(torch.empty(0, 192, dtype=torch.bfloat16, device=dev), 1, 1, 64, none, k, v, ks, vs, 16)
    assert paged.page_gather(k, v, ks, vs, none, 1, 64, 16).shape == (0, 128)
    out = paged.page_attention(torch.empty(0, 64, dtype=torch.bfloat16, device=dev), k, v, ks, vs,
                               torch.empty(0, 3, dtype=torch.int32, device=dev), none, 16, 1, 1, 64)
    assert out.shape == (0, 64)
    paged.copy_pages([k[None]], [], 2)
    # a table without columns: no page to read
    out = paged.page_attention(torch.ones(1, 64, dtype=torch.bfloat16, device=dev), k, v, ks, vs,
                               torch.empty(1, 0, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev), 16, 1, 1, 64)
    assert not out.any() and _status_code() == ""


# ------------------------------------------------------------------ page copies
@pytest.mark.parametrize("layers,pages,shapes", [
    (3, 20, [(16, 2, 64, torch.bfloat16)] * 2),
    (2, 33, [(7, 3, 64, torch.float8_e4m3fn), (7, 3, 64, torch.float8_e4m3fn), (1, 3, 1, torch.float32), (1, 3, 1, torch.float32)]),
    (1, 50, [(1, 1, 3, torch.int8), (1, 1, 5, torch.float32), (3, 1, 1, torch.bfloat16)]),
    (5, 9, [(64, 8, 128, torch.float32)])])
def test_copy_pages(layers, pages, shapes):
    g = torch.Generator(device=dev).manual_seed(1)
    caches = []
    for rows, h, d, dt in shapes:
        n = layers * pages * rows * h * d * torch.empty(0, dtype=dt).element_size()
        b = torch.randint(0, 256, (n,), device=dev, generator=g, dtype=torch.int32).to(torch.uint8)
        caches.append(b.view(dt).view(layers, pages * rows, h, d))
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).tolist()
    n = pages // 3
    moves = list(zip(order[:n] + order[:1], order[n:2 * n + 1]))  # one page forked twice
    for as_list in (True, False):
        got = [c.clone() for c in caches]
        P().copy_pages(got, moves if as_list else torch.tensor(moves, dtype=torch.int32, device=dev), pages)
        for a, c, (rows, h, d, dt) in zip(got, caches, shapes):
            want = c.view(torch.uint8).view(layers, pages, -1).clone()
            for s, t in moves:
                want[:, t] = want[:, s]
            assert torch.equal(a.view(torch.uint8).view(layers, pages, -1), want)
    assert _status_code() == ""


def test_copy_pages_refuses():
    c = torch.zeros(2, 8, 4, device=dev)
    for moves in ([(0, 1), (2, 1)], [(0, 1), (1, 2)], [(3, 3)], [(0, 8)], [(-1, 2)]):
        with pytest.raises(ValueError):
            P().copy_pages([c], moves, 8)
    with pytest.raises(RuntimeError):
        P().copy_pages([c], [(0, 1)], 3)  # 8 rows are not 3 pages
    with pytest.raises(RuntimeError):
        P().copy_pages([c] * 9, [(0, 1)], 8)
    with pytest.raises(RuntimeError):
        P().copy_pages([c, torch.zeros(3, 8, 4, device=dev)], [(0, 1)], 8)
    c += torch.arange(8, device=dev)[None, :, None]
    P().copy_pages([c], torch.tensor([[0, 8], [1, 2], [-1, 3], [4, 1 << 30]], dtype=torch.int32, device=dev), 8)
    assert "out of range" in _status_code()
    assert c[0, :, 0].tolist() == [0, 1, 1, 3, 4, 5, 6, 7]


# ------------------------------------------------------------------ refusals
def test_counts_past_31_bits_are_refused():
    """Rows, moves, histories and biases whose indexes would pass 31 bits (nothing is launched; 17 GB, never touched)."""
    from lora_kernel_b200.ops import logits
    paged = P()
    k, v, ks, vs = _cache("fp8_page", 2, 16, 1, 64)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    tokens = torch.empty(2 ** 31, dtype=torch.int64, device=dev)
    out = torch.empty(1, 128, dtype=torch.bfloat16, device=dev)
    slots = tokens.view(torch.int32)
    for n in (2 ** 28 - 1, 2 ** 31 - 4096, 2 ** 31, 2 ** 32):  # the first: items of the last block alone pass 31 bits
        with pytest.raises(RuntimeError):
            paged.page_gather(k, v, ks, vs, slots[:n], 1, 64, 16, out=out.expand(n, 128))
    with pytest.raises(RuntimeError):
        paged.copy_pages([k[None]], slots.view(-1, 2), 2)
    counts = torch.zeros(2, 64, dtype=torch.int16, device=dev)
    with pytest.raises(RuntimeError):
        logits.set_token_counts(counts, None, tokens, i32(2), i32(1))
    with pytest.raises(RuntimeError):
        logits.add_token_counts(counts, slots[:2 ** 31], tokens)
    with pytest.raises(RuntimeError):
        logits.adjust_logits(torch.zeros(1, 64, device=dev), bias=(i32(2), slots[:2 ** 31], slots[:2 ** 31].view(torch.float32)))
    del tokens, slots
    torch.cuda.empty_cache()


def test_tables_of_too_many_tokens_are_refused():
    """Whatever max_ctx says: a context's end near 2^31 would take token indexes past it."""
    paged = P()
    none = torch.empty(0, dtype=torch.int32, device=dev)
    q = torch.empty(0, 64, dtype=torch.bfloat16, device=dev)
    for page, width in ((1, 2 ** 31 - 8), (16, 2 ** 27), (64, 2 ** 40)):
        k, v, ks, vs = _cache("fp8_page", 2, page, 1, 64)
        for max_ctx in (0, 5):
            with pytest.raises(RuntimeError, match="block_tables"):
                paged.page_attention(q, k, v, ks, vs, torch.empty(0, width, dtype=torch.int32, device=dev), none, page, 1, 1, 64, max_ctx=max_ctx)
        out = paged.page_attention(q, k, v, ks, vs, torch.empty(0, 2 ** 20, dtype=torch.int32, device=dev), none, page, 1, 1, 64, max_ctx=5)
        assert out.shape == (0, 64)


def test_refusals():
    paged = P()
    Hq, Hkv, Dh, page = 4, 2, 64, 16
    k, v, ks, vs = _cache("fp8_page", 4, page, Hkv, Dh)
    qkv = torch.zeros(2, (Hq + 2 * Hkv) * Dh, dtype=torch.bfloat16, device=dev)
    slots = torch.zeros(2, dtype=torch.int32, device=dev)
    ok = dict(qkv=qkv, slots=slots, k=k, v=v, ks=ks, vs=vs, page=page, Dh=Dh)

    def append(**kw):
        a = {**ok, **kw}
        paged.page_append(a["qkv"], Hq, Hkv, a["Dh"], a["slots"], a["k"], a["v"], a["ks"], a["vs"], a["page"])

    def attend(**kw):
        a = {**dict(q=qkv[:, :Hq * Dh], bt=torch.zeros(2, 1, dtype=torch.int32, device=dev),
                    ctx=torch.ones(2, dtype=torch.int32, device=dev), Hq=Hq, q_len=1), **ok, **kw}
        return paged.page_attention(a["q"], a["k"], a["v"], a["ks"], a["vs"], a["bt"], a["ctx"], a["page"], a["Hq"], Hkv, a["Dh"],
                                    q_len=a["q_len"], out=a.get("out"))

    bad = [dict(qkv=qkv.float()), dict(qkv=qkv[:, 1:]), dict(slots=slots.long()), dict(slots=slots[:1]), dict(k=k.view(torch.int8)),
           dict(k=k.float(), v=v.float()), dict(ks=ks[:2]), dict(vs=vs.half()), dict(page=3), dict(Dh=32), dict(ks=ks.cpu())]
    for kw in bad:
        with pytest.raises(RuntimeError):
            append(**kw)
    bad = [dict(q=qkv), dict(q=qkv[:, :Hq * Dh].float()), dict(q=qkv[:, 4:4 + Hq * Dh]), dict(bt=torch.zeros(3, 1, dtype=torch.int32, device=dev)),
           dict(bt=torch.zeros(2, 1, dtype=torch.int64, device=dev)), dict(ctx=torch.ones(1, dtype=torch.int32, device=dev)), dict(Hq=3),
           dict(q_len=0), dict(q_len=3), dict(out=torch.empty(2, Hq * Dh, device=dev)), dict(out=torch.empty(1, Hq * Dh, dtype=torch.bfloat16, device=dev)),
           dict(page=5), dict(v=v[:16])]
    for kw in bad:
        with pytest.raises(RuntimeError):
            attend(**kw)
    with pytest.raises(RuntimeError):
        paged.page_gather(k, v, ks, vs, slots, Hkv, Dh, page, out=torch.empty(2, 8, dtype=torch.bfloat16, device=dev))
    with pytest.raises(RuntimeError):
        paged.page_append(qkv.cpu(), Hq, Hkv, Dh, slots, k, v, ks, vs, page)
    with pytest.raises(KeyError):
        paged.new_page_cache(1, 4, 16, 2, 64, "fp8")
    append()
    attend()
