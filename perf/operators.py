"""Cases of the serving operators over the page-scaled 8-bit KV cache: appending to it and reading it back, attention
over it, copying its pages, and the logits' penalties, biases and grammar masks.

Sequence lengths, page tables and history lengths are functions of the case alone (so that work() knows them); the
values are made from the seed."""
import functools
import math

import torch

own = False
dev = "cuda"

QMAX = {"fp8": 448.0, "int8": 127.0}
CODE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
HALF = {"bf16": torch.bfloat16, "f32": torch.float32}


@functools.lru_cache(None)
def _package():
    from lora_kernel_b200.ops import logits, paged
    return paged, logits


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the first decode steps of one request to the small test model: what a launch costs
        {"name": "attend_first", "op": "attend", "n": 1, "q_len": 1, "hq": 4, "hkv": 2, "dh": 64, "page": 16, "ctx": 33, "kind": "fp8"},
        # a server's full decode batch, contexts of every length up to the longest
        {"name": "attend_batch", "op": "attend", "n": 256, "q_len": 1, "hq": 32, "hkv": 8, "dh": 128, "page": 16, "ctx": 4096, "kind": "fp8"},
        # draft tokens verified together (speculative decoding), int8 pages of an odd size
        {"name": "attend_verify", "op": "attend", "n": 24, "q_len": 5, "hq": 32, "hkv": 4, "dh": 64, "page": 24, "ctx": 2047, "kind": "int8"},
        # two long documents: few rows, the work has to be split along the context
        {"name": "attend_long", "op": "attend", "n": 2, "q_len": 1, "hq": 32, "hkv": 8, "dh": 128, "page": 32, "ctx": 100003, "kind": "fp8"},
        # a few tokens after a prompt that ended inside a page
        {"name": "append_few", "op": "append", "n": 2, "new": 5, "hq": 4, "hkv": 2, "dh": 64, "page": 24, "start": 31, "kind": "int8"},
        # one token for each sequence of a full decode batch
        {"name": "append_decode", "op": "append", "n": 256, "new": 1, "hq": 32, "hkv": 8, "dh": 128, "page": 16, "start": 1000, "kind": "fp8"},
        # a whole prefill budget: chunks of prompts that go on where the last chunk stopped, read back for the prefill attention
        {"name": "append_prefill", "op": "append", "n": 3, "new": 2730, "hq": 32, "hkv": 8, "dh": 128, "page": 16, "start": 1301, "kind": "fp8"},
        # one sequence forked into four continuations: its partly filled page in every layer
        {"name": "pages_fork", "op": "pages", "layers": 32, "pairs": 3, "pages": 64, "page": 16, "hkv": 8, "dh": 128, "kind": "bf16"},
        # compaction after most requests ended: the scattered pages move to the front
        {"name": "pages_compact", "op": "pages", "layers": 22, "pairs": 1500, "pages": 4096, "page": 16, "hkv": 4, "dh": 64, "kind": "bf16"},
        # one request with penalties
        {"name": "logits_one", "op": "logits", "n": 1, "vocab": 32000, "kind": "bf16", "history": 0, "bias": 0, "mask": False},
        # a full decode batch with penalties, biases and grammars
        {"name": "logits_batch", "op": "logits", "n": 256, "vocab": 128256, "kind": "bf16", "history": 0, "bias": 300, "mask": True},
        # requests admitted again: their counts built from their histories, then the logits; an odd vocabulary
        {"name": "logits_admit", "op": "logits", "n": 48, "vocab": 32003, "kind": "f32", "history": 3000, "bias": 17, "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "pages", "logits", "logits"])
    kind = rng.choice(["fp8", "fp8", "int8"])
    page = rng.choice([16, 16, 32, rng.randint(1, 64)])
    dh = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 4, 7, 8])
    if op == "attend":
        n, q_len = _log(rng, 1, 256), rng.choice([1, 1, 1, rng.randint(2, 8)])
        most = min(131072, max(16, int(1.0e9 / (n * 2 * hkv * dh))))
        return {"op": op, "n": n, "q_len": q_len, "hq": hkv * group, "hkv": hkv, "dh": dh, "page": page, "ctx": _log(rng, 1, most), "kind": kind}
    if op == "append":
        n = _log(rng, 1, 256)
        return {"op": op, "n": n, "new": _log(rng, 1, max(1, 8192 // n)), "hq": hkv * group, "hkv": hkv, "dh": dh, "page": page,
                "start": _log(rng, 1, min(4096, 30000 // n)) - 1, "kind": kind}
    if op == "pages":
        layers, page = rng.randint(1, 32), min(page, 32)
        pages = _log(rng, 16, max(16, min(4096, 2 ** 28 // (layers * page * hkv * dh))))
        return {"op": op, "layers": layers, "pairs": _log(rng, 1, pages // 3), "pages": pages, "page": page, "hkv": hkv, "dh": dh,
                "kind": rng.choice(["bf16", "bf16", "f32"])}
    n = _log(rng, 1, 256)
    return {"op": op, "n": n, "vocab": _log(rng, 1000, min(128256, 2 ** 25 // n)), "kind": rng.choice(["bf16", "bf16", "f32"]),
            "history": rng.choice([0, 0, _log(rng, 1, 4000)]), "bias": rng.choice([0, rng.randint(1, 300)]), "mask": rng.choice([True, False])}


def _ragged(n, most):
    """n lengths in [0, most], the first of them `most`; an unused batch row (0) where there are several."""
    got = [most] + [int(most * math.modf(i * 0.6180339887)[0]) + 1 for i in range(1, n)]
    if n > 3:
        got[2] = 0
    return [min(x, most) for x in got]


# ------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    made = {"attend": _prepare_attend, "append": _prepare_append, "pages": _prepare_pages, "logits": _prepare_logits}[case["op"]](case, g)
    return dict(case, **made)


def _pow2_scale(amax, qmax):
    """The smallest power of two s with amax <= qmax * s (at least 2^-126)."""
    frac, exp = torch.frexp(amax / qmax)
    exp = torch.where(frac == 0.5, exp - 1, exp)
    exp = torch.where(amax > 0, exp, torch.full_like(exp, -126)).clamp(-126, 127)
    return torch.ldexp(torch.ones_like(amax), exp)


def _round(x, kind):
    """x (already divided by the scale) rounded to the codes' values."""
    return x.to(torch.float8_e4m3fn) if kind == "fp8" else x.round().to(torch.int8)


def _filled_cache(case, pages, g):
    """A cache of `pages` full pages: codes [slots, Hkv, Dh] and scales [pages, Hkv], keys with a few large channels."""
    page, hkv, dh, kind = case["page"], case["hkv"], case["dh"], case["kind"]
    made = []
    for which in range(2):
        x = torch.randn(pages, page, hkv, dh, device=dev, generator=g)
        x *= torch.rand(hkv, dh, device=dev, generator=g).pow(8) * 6 + 0.5 if which == 0 else 0.7
        scale = _pow2_scale(x.abs().amax(dim=(1, 3)), QMAX[kind])
        x /= scale[:, None, :, None]
        made += [_round(x, kind).view(pages * page, hkv, dh), scale]
    return made


def _tables(lens, page, total, g):
    """Page table [n, most pages] (int32) of sequences of these lengths over `total` pages in random order."""
    need = torch.tensor([-(-x // page) for x in lens])
    most = max(1, int(need.max()))
    order = torch.randperm(total, device=dev, generator=g).to(torch.int32)
    col = torch.arange(most)[None, :]
    at = (need.cumsum(0) - need)[:, None] + col
    table = order[at.clamp(max=total - 1).to(dev)]
    table[(col >= need[:, None]).to(dev)] = 0
    return table.contiguous()


def _prepare_attend(case, g):
    lens = _ragged(case["n"], case["ctx"])
    total = sum(-(-x // case["page"]) for x in lens) + 3
    kc, ks, vc, vs = _filled_cache(case, total, g)
    heads = case["hq"] + 2 * case["hkv"]
    qkv = torch.randn(case["n"] * case["q_len"], heads * case["dh"], device=dev, generator=g).to(torch.bfloat16)
    return {"qkv": qkv, "kc": kc, "ks": ks, "vc": vc, "vs": vs, "tables": _tables(lens, case["page"], total, g),
            "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}


def _starts(case):
    """Tokens that each sequence has in the cache before the call."""
    return [max(0, case["start"] - 7 * i) if case["new"] > 1 else case["start"] + i for i in range(case["n"])]


def _read_back(case):
    """Where each sequence's values are read back from: the whole context for a chunk of a prompt, the last page for one token."""
    return [0 if case["new"] > 1 else s - s % case["page"] for s in _starts(case)]


def _prepare_append(case, g):
    page, new, starts = case["page"], case["new"], _starts(case)
    lens = [s + new for s in starts]
    total = sum(-(-x // page) for x in lens) + 3
    kc, ks, vc, vs = _filled_cache(case, total, g)
    table = _tables(lens, page, total, g).long()

    def slots(begin, end):
        seq = torch.cat([torch.full((b - a,), i) for i, (a, b) in enumerate(zip(begin, end))]).to(dev)
        pos = torch.cat([torch.arange(a, b) for a, b in zip(begin, end)]).to(dev)
        return (table[seq, pos // page] * page + pos % page).to(torch.int32)

    heads = case["hq"] + 2 * case["hkv"]
    qkv = torch.randn(case["n"] * new, heads * case["dh"], device=dev, generator=g)
    qkv *= torch.rand(case["n"] * new, 1, device=dev, generator=g) * 3 + 0.5
    return {"qkv": qkv.to(torch.bfloat16), "kc": kc, "ks": ks, "vc": vc, "vs": vs, "slots": slots(starts, lens),
            "back": slots(_read_back(case), lens)}


def _prepare_pages(case, g):
    shape = (case["layers"], case["pages"] * case["page"], case["hkv"], case["dh"])
    kc, vc = (torch.randn(shape, device=dev, generator=g, dtype=HALF[case["kind"]]) for _ in range(2))
    order = torch.randperm(case["pages"], device=dev, generator=g)[: 2 * case["pairs"]].to(torch.int32)
    return {"kc": kc, "vc": vc, "moves": order.view(2, -1).t().contiguous()}


def _prepare_logits(case, g):
    n, vocab = case["n"], case["vocab"]
    logits = (torch.randn(n, vocab, device=dev, generator=g) * 3).to(HALF[case["kind"]])
    rows = torch.randperm(n + 2, device=dev, generator=g)[:n].to(torch.int32)  # the requests' rows of the server's table
    pick = torch.rand(n, 3, device=dev, generator=g)
    penalties = torch.stack([1 + pick[:, 0] * 0.5, pick[:, 1] - 0.2, pick[:, 2] - 0.2], dim=1)
    penalties[:: 3, 0] = 1.0
    made = {"logits": logits, "rows": rows, "penalties": penalties.contiguous(), "tokens": None, "offsets": None, "prompts": None,
            "bias": None, "mask": None, "mask_rows": None}
    made["counts"] = torch.zeros(n + 2, vocab, dtype=torch.int16, device=dev)
    if case["history"]:
        sizes = torch.tensor(_ragged(n, case["history"]))
        made["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).to(torch.int32).to(dev)
        made["tokens"] = (torch.rand(int(sizes.sum()), device=dev, generator=g).pow(3) * vocab).long().clamp(max=vocab - 1)
        made["prompts"] = (sizes * 2 // 3).to(torch.int32).to(dev)
    else:  # a history of up to 1000 tokens already counted
        seen = torch.rand(n + 2, vocab, device=dev, generator=g) * vocab
        made["counts"] += (seen < 300).to(torch.int16) + 3 * (seen < 40).to(torch.int16)
        made["counts"][(seen > 200) & (seen < 900)] += -32768
    if case["bias"]:
        each = min(case["bias"], vocab)
        step = vocab // each
        ids = (torch.arange(each, device=dev) * step)[None] + torch.randint(0, step, (n, 1), device=dev, generator=g)
        made["bias"] = (torch.arange(n + 1, dtype=torch.int32, device=dev) * each, ids.reshape(-1).to(torch.int32),
                        torch.randn(n * each, device=dev, generator=g) * 5)
    if case["mask"]:
        words = (vocab + 31) // 32
        made["mask"] = torch.randint(-2 ** 31, 2 ** 31, (n, words), device=dev, generator=g).to(torch.int32)
        made["mask"][:: 2] &= torch.randint(-2 ** 31, 2 ** 31, (n, words), device=dev, generator=g).to(torch.int32)[:: 2]
        made["mask_rows"] = torch.arange(n, dtype=torch.int32, device=dev).flip(0)
        made["mask_rows"][:: 4] = -1  # requests without a grammar
    return made


# ------------------------------------------------------------------ one pass
def run(s):
    return {"attend": _attend, "append": _append, "pages": _pages, "logits": _logits}[s["op"]](s)


def _attend(s):
    q = s["qkv"][:, : s["hq"] * s["dh"]]
    if own:
        paged, _ = _package()
        return paged.page_attention(q, s["kc"], s["vc"], s["ks"], s["vs"], s["tables"], s["lens"], s["page"], s["hq"], s["hkv"], s["dh"],
                                    q_len=s["q_len"], max_ctx=s["ctx"])
    n, q_len, hkv, dh, page = s["n"], s["q_len"], s["hkv"], s["dh"], s["page"]
    group = s["hq"] // hkv
    table = s["tables"].long()
    most = table.shape[1] * page

    def values(codes, scale):  # [n, Hkv, tokens, Dh]
        x = codes.view(-1, page, hkv, dh)[table].float() * scale[table][:, :, None, :, None]
        return x.reshape(n, most, hkv, dh).transpose(1, 2)

    pos = torch.arange(most, device=dev)
    there = pos[None, :] < s["lens"][:, None]
    last = s["lens"][:, None] - q_len + torch.arange(q_len, device=dev)[None, :]  # [n, q_len]: each query's own position
    seen = pos[None, None, :] <= last[:, :, None]
    qf = q.float().reshape(n, q_len, hkv, group, dh).permute(0, 2, 1, 3, 4).reshape(n, hkv, q_len * group, dh)
    score = (qf @ values(s["kc"], s["ks"]).transpose(-1, -2)) / math.sqrt(dh)
    seen = seen[:, None, :, None, :].expand(n, 1, q_len, group, most).reshape(n, 1, q_len * group, most)
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    v = torch.where(there[:, None, :, None], values(s["vc"], s["vs"]), torch.zeros((), device=dev))
    out = (p @ v) / p.sum(dim=-1, keepdim=True).clamp(min=1e-37)
    return out.view(n, hkv, q_len, group, dh).permute(0, 2, 1, 3, 4).reshape(n * q_len, s["hq"] * dh).to(torch.bfloat16)


def _append(s):
    if own:
        paged, _ = _package()
        paged.page_append(s["qkv"], s["hq"], s["hkv"], s["dh"], s["slots"], s["kc"], s["vc"], s["ks"], s["vs"], s["page"])
        back = paged.page_gather(s["kc"], s["vc"], s["ks"], s["vs"], s["back"], s["hkv"], s["dh"], s["page"])
        return {"back": back, "ks": s["ks"], "vs": s["vs"]}
    hkv, dh, page, kind, slots = s["hkv"], s["dh"], s["page"], s["kind"], s["slots"].long()
    pages, at = torch.unique(slots // page, return_inverse=True)
    first = torch.full_like(pages, page).scatter_reduce(0, at, slots % page, "amin")  # the first new offset in each page
    kept = torch.arange(page, device=dev)[None, :] < first[:, None]
    rows = s["qkv"].float().view(-1, s["hq"] + 2 * hkv, dh)

    def put(x, codes, scale):
        top = torch.zeros(pages.numel(), hkv, device=dev).scatter_reduce(0, at[:, None].expand(-1, hkv), x.abs().amax(dim=-1), "amax")
        old = scale[pages]
        now = _pow2_scale(top, QMAX[kind])
        now = torch.where((first > 0)[:, None], torch.maximum(old, now), now)
        held = codes.view(-1, page, hkv, dh)[pages]
        moved = _round(held.float() * (old / now)[:, None, :, None], kind)
        same = kept[:, :, None, None] & (old < now)[:, None, :, None]
        codes.view(-1, page, hkv, dh)[pages] = torch.where(same, moved.view(torch.int8), held.view(torch.int8)).view(codes.dtype)
        codes[slots] = _round(x / now[at][:, :, None], kind)
        scale[pages] = now

    put(rows[:, s["hq"]:s["hq"] + hkv], s["kc"], s["ks"])
    put(rows[:, s["hq"] + hkv:], s["vc"], s["vs"])
    back = s["back"].long()
    key = s["kc"][back].float() * s["ks"][back // page][:, :, None]
    value = s["vc"][back].float() * s["vs"][back // page][:, :, None]
    return {"back": torch.stack([key, value], dim=1).reshape(back.numel(), 2 * hkv * dh).to(torch.bfloat16), "ks": s["ks"], "vs": s["vs"]}


def _pages(s):
    if own:
        paged, _ = _package()
        paged.copy_pages([s["kc"], s["vc"]], s["moves"], s["pages"])
        return s["kc"], s["vc"]
    src, dst = s["moves"][:, 0].long(), s["moves"][:, 1].long()
    shape = (s["layers"], s["pages"], s["page"] * s["hkv"] * s["dh"])
    s["kc"].view(shape)[:, dst] = s["kc"].view(shape)[:, src]
    s["vc"].view(shape)[:, dst] = s["vc"].view(shape)[:, src]
    return s["kc"], s["vc"]


def _logits(s):
    if own:
        _, ops = _package()
        if s["tokens"] is not None:
            ops.set_token_counts(s["counts"], s["rows"], s["tokens"], s["offsets"], s["prompts"])
        z = ops.adjust_logits(s["logits"], s["counts"], s["rows"], s["penalties"], bias=s["bias"], mask=s["mask"], mask_rows=s["mask_rows"])
        return {"logits": z, "counts": s["counts"]} if s["tokens"] is not None else {"logits": z}
    n, vocab = s["logits"].shape
    rows = s["rows"].long()
    if s["tokens"] is not None:
        size = s["offsets"].diff()
        row = torch.repeat_interleave(torch.arange(n, device=dev), size.long(), output_size=s["tokens"].numel())
        prompt = torch.arange(s["tokens"].numel(), device=dev) - s["offsets"][row] < s["prompts"][row]
        flag = torch.zeros(n, vocab, dtype=torch.int32, device=dev)
        flag.index_put_((row, s["tokens"]), prompt.int(), accumulate=True)
        count = torch.zeros(n, vocab, dtype=torch.int32, device=dev)
        count.index_put_((row, s["tokens"]), (~prompt).int(), accumulate=True)
        s["counts"][rows] = (count.clamp(max=32767) - 32768 * (flag > 0).int()).to(torch.int16)
    held = s["counts"][rows].int()
    count = held & 0x7FFF
    z = s["logits"].float()
    r, f, p = (s["penalties"][:, i:i + 1] for i in range(3))
    z = torch.where(held != 0, torch.where(z > 0, z / r, z * r), z)
    z = z - f * count - p * (count > 0)
    if s["bias"] is not None:
        offsets, ids, values = s["bias"]
        row = torch.repeat_interleave(torch.arange(n, device=dev), offsets.diff().long(), output_size=ids.numel())
        z.index_put_((row, ids.long()), values, accumulate=True)
    if s["mask"] is not None:
        which = s["mask_rows"].long()
        bits = (s["mask"][which.clamp(min=0)][:, :, None] >> torch.arange(32, device=dev, dtype=torch.int32)) & 1
        allowed = (bits.reshape(n, -1)[:, :vocab] != 0) | (which < 0)[:, None]
        z = torch.where(allowed, z, torch.full_like(z, -math.inf))
    z = z.to(s["logits"].dtype)
    return {"logits": z, "counts": s["counts"]} if s["tokens"] is not None else {"logits": z}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "attend":
        lens, row = _ragged(c["n"], c["ctx"]), c["hkv"] * c["dh"]
        pages = sum(-(-x // c["page"]) for x in lens)
        data = sum(lens) * 2 * row + pages * c["hkv"] * 8 + 2 * c["n"] * c["q_len"] * c["hq"] * c["dh"] * 2
        return {"bytes": data, "flops": 4 * sum(lens) * c["q_len"] * c["hq"] * c["dh"]}
    if c["op"] == "append":
        row = 2 * c["hkv"] * c["dh"]
        back = sum(s + c["new"] - b for s, b in zip(_starts(c), _read_back(c)))
        return {"bytes": c["n"] * c["new"] * row * 3 + back * row * 3, "flops": c["n"] * c["new"] * row * 3 + back * row}
    if c["op"] == "pages":
        size = c["page"] * c["hkv"] * c["dh"] * (2 if c["kind"] == "bf16" else 4)
        return {"bytes": 4 * c["pairs"] * c["layers"] * size, "flops": 0}
    each = 2 if c["kind"] == "bf16" else 4
    data = c["n"] * c["vocab"] * (2 * each + 2) + c["n"] * c["bias"] * 8
    if c["history"]:
        data += c["n"] * c["vocab"] * 2 + sum(_ragged(c["n"], c["history"])) * 8
    if c["mask"]:
        data += c["n"] * ((c["vocab"] + 31) // 32) * 4
    return {"bytes": data, "flops": 5 * c["n"] * c["vocab"]}


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    """What run() returns for these inputs, computed in 64 bits."""

    def attend(s):
        """Sequence by sequence and head by head."""
        q_len, hq, hkv, dh, page = s["q_len"], s["hq"], s["hkv"], s["dh"], s["page"]
        out = torch.zeros(s["n"], q_len, hq, dh, dtype=torch.float64, device=dev)
        q = s["qkv"][:, : hq * dh].double().view(s["n"], q_len, hq, dh)
        for i, ctx in enumerate(s["lens"].tolist()):
            if ctx == 0:
                continue
            ids = s["tables"][i, : -(-ctx // page)].long()
            k = (s["kc"].view(-1, page, hkv, dh)[ids].double() * s["ks"].double()[ids][:, None, :, None]).flatten(0, 1)[:ctx]
            v = (s["vc"].view(-1, page, hkv, dh)[ids].double() * s["vs"].double()[ids][:, None, :, None]).flatten(0, 1)[:ctx]
            for j in range(q_len):
                upto = ctx - q_len + j + 1
                if upto <= 0:
                    continue
                kj, vj = (x[:upto].repeat_interleave(hq // hkv, dim=1) for x in (k, v))
                p = torch.softmax(torch.einsum("hd,thd->ht", q[i, j], kj) / math.sqrt(dh), dim=-1)
                out[i, j] = torch.einsum("ht,thd->hd", p, vj)
        return out.view(s["n"] * q_len, hq * dh)

    def nearest(x, kind):
        """x rounded to the nearest value of the type, ties to even (x within the type's range)."""
        if kind == "int8":
            return torch.round(x)
        exp = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)) + 1e-9)  # log2 of a power of two may come out an ulp low
        unit = torch.exp2(exp - 3)  # spacing: 3 bits after the leading one, at least 2^-9
        return torch.round(x / unit) * unit

    def append(s):
        """Page by page, in the order of the rows."""
        hq, hkv, dh, page, kind = s["hq"], s["hkv"], s["dh"], s["page"], s["kind"]
        rows = s["qkv"].double().view(-1, hq + 2 * hkv, dh)
        slots = s["slots"].tolist()
        runs, t = [], 0
        while t < len(slots):
            e = t + 1
            while e < len(slots) and slots[e] // page == slots[t] // page:
                e += 1
            runs.append((t, e))
            t = e
        if len(runs) > 3000:
            return None
        sides = []
        for at, codes, scale in ((hq, s["kc"], s["ks"]), (hq + hkv, s["vc"], s["vs"])):
            codes, scale = codes.double(), scale.double()
            top = rows[:, at:at + hkv].abs().amax(dim=-1)
            for t, e in runs:
                p, a = slots[t] // page, slots[t] % page
                need = torch.log2(top[t:e].amax(dim=0) / QMAX[kind])
                now = torch.exp2(torch.ceil(need - 1e-9).clamp(min=-126))  # bf16 maxima are further apart than this
                if a > 0:
                    now = torch.maximum(now, scale[p])
                    held = codes[p * page: p * page + a]
                    held.copy_(nearest(held * (scale[p] / now)[None, :, None], kind))
                codes[slots[t]: slots[t] + e - t] = nearest(rows[t:e, at:at + hkv] / now[None, :, None], kind)
                scale[p] = now
            back = s["back"].long()
            sides += [codes[back] * scale[back // page][:, :, None], scale]
        return {"back": torch.stack([sides[0], sides[2]], dim=1).reshape(-1, 2 * hkv * dh), "ks": sides[1], "vs": sides[3]}

    def pages(s):
        """Each page's contents after the moves."""
        of = torch.arange(s["pages"], device=dev)
        of[s["moves"][:, 1].long()] = s["moves"][:, 0].long()
        return tuple(c.unflatten(1, (s["pages"], s["page"])).index_select(1, of).flatten(1, 2).double() for c in (s["kc"], s["vc"]))

    def logits(s):
        """Row by row."""
        n, vocab = s["logits"].shape
        counts = s["counts"].clone()
        out = s["logits"].double()
        for i, row in enumerate(s["rows"].tolist()):
            if s["tokens"] is not None:
                a, b = s["offsets"][i].item(), s["offsets"][i + 1].item()
                cut = a + s["prompts"][i].item()
                made = torch.bincount(s["tokens"][cut:b], minlength=vocab).clamp(max=32767)
                made[s["tokens"][a:cut].unique()] -= 32768
                counts[row] = made.to(torch.int16)
            held = counts[row].long()
            r, f, p = s["penalties"][i].double().tolist()
            z = out[i]
            z[:] = torch.where(held == 0, z, torch.where(z > 0, z / r, z * r))
            count = torch.where(held < 0, held + 32768, held)
            z -= f * count + p * (count > 0)
            if s["bias"] is not None:
                offsets, ids, values = s["bias"]
                a, b = offsets[i].item(), offsets[i + 1].item()
                z.index_add_(0, ids[a:b].long(), values[a:b].double())
            if s["mask"] is not None and s["mask_rows"][i].item() >= 0:
                token = torch.arange(vocab, device=dev)
                word = s["mask"][s["mask_rows"][i].item()][token // 32].long()
                z[(word >> (token % 32)) & 1 == 0] = -math.inf
        return {"logits": out, "counts": counts} if s["tokens"] is not None else {"logits": out}

    return {"attend": attend, "append": append, "pages": pages, "logits": logits}[case["op"]](prepare(case, seed))
