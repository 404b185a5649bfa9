"""Forks, several samples, compaction, penalties and grammars in the engine, on CPU: a fake runner keeps a token-level
KV store that page copies move about, so that a wrong block, a missing copy or a stale count changes the output."""
import random

import pytest
import torch

from lora_kernel_b200.config import ServeConfig, TransformerConfig
from lora_kernel_b200.serve.engine import LLMEngine, SamplingParams
from lora_kernel_b200.serve.kv_cache import BlockManager
from lora_kernel_b200.serve.security import InputValidator, ValidationError
from paged_oracle import adjust, token_counts
from test_engine_cpu import KVRunner, V, next_token, reference


class Runner(KVRunner):
    """KVRunner with page copies, and logits changes by the 64-bit oracle."""

    supports_adjust = True
    supports_top_p = True

    def __init__(self, *a):
        super().__init__(*a)
        self.counts, self.copied = {}, []

    def copy_pages(self, moves):
        bs = self.block_size
        before = dict(self.kv)
        assert len({d for _, d in moves}) == len(moves) and not {d for _, d in moves} & {s for s, _ in moves}
        for s, d in moves:
            self.copied.append((s, d))
            for k in range(bs):
                if s * bs + k in before:
                    self.kv[d * bs + k] = before[s * bs + k]

    def set_counts(self, rows, histories, table_rows):
        for r, (p, o) in zip(rows, histories):
            assert r < table_rows
            self.counts[r] = token_counts(p, o, V)

    def add_counts(self, rows, tokens):
        for r, t in zip(rows, tokens.tolist()):
            if r >= 0:
                self.counts[r][t] += 1

    def adjust_logits(self, logits, rows, penalties, biases, allowed):
        out = []
        for k, r in enumerate(rows):
            a = None
            if allowed[k] is not None:
                a = torch.zeros(V, dtype=torch.bool)
                a[list(allowed[k])] = True
            out.append(adjust(logits[k].double(), self.counts[r] if r >= 0 else None, penalties[k], biases[k], a))
        return torch.stack(out)

    def _logits(self, ctx):
        # a soft ranking: the next token first, then the tokens after it
        z = torch.arange(V, 0, -1).float()
        return z.roll(next_token(ctx)) / 10

    def sample(self, logits, temps, seed, top_ps=None, row_seeds=None):
        return torch.argmax(logits, dim=-1)


def _engine(num_blocks=64, block_size=4, cls=Runner, **kw):
    sc = ServeConfig(num_kv_blocks=num_blocks, block_size=block_size, cuda_graphs=False, max_model_len=512, **kw)
    runner = cls(num_blocks, block_size)
    return LLMEngine(TransformerConfig(vocab_size=V), None, sc, runner=runner), runner


def _run(eng, ids):
    while any(i not in eng.finished for i in ids):
        eng.step()


def _penalised(prompt, n, p):
    """The engine's greedy output with these parameters, one token after another."""
    out = []
    soft = Runner(1, 1)
    while len(out) < n:
        ok = p.allowed(out)
        if ok is not None and not len(ok):
            break
        mask = None
        if ok is not None:
            mask = torch.zeros(V, dtype=torch.bool)
            mask[list(ok)] = True
        c = token_counts(prompt, out, V) if p.penalised else None
        z = adjust(soft._logits(prompt + out).double(), c, (p.repetition_penalty, p.frequency_penalty, p.presence_penalty), p.logit_bias, mask)
        out.append(int(torch.argmax(z)))
    return out


# ------------------------------------------------------------------ blocks
def test_fork_shares_full_blocks_and_copies_the_tail():
    bm = BlockManager(8, 4)
    table, _ = bm.allocate(list(range(10)))
    child, copies = bm.fork(table, 10)
    assert child[:2] == table[:2] and child[2] != table[2] and copies == [(table[2], child[2])]
    assert [bm.ref[b] for b in table] == [2, 2, 1]
    even, none = bm.fork(table, 8)
    assert even == table[:2] and none == []
    bm.free_seq(table)
    bm.free_seq(even)
    assert bm.ref[child[0]] == 1 and bm.num_free() == 8 - 3
    bm.free_seq(child)
    assert bm.num_free() == 8


def test_fork_without_a_free_block_changes_nothing():
    bm = BlockManager(3, 4)
    table, _ = bm.allocate(list(range(10)))
    ref = list(bm.ref)
    with pytest.raises(MemoryError):
        bm.fork(table, 9)
    assert bm.ref == ref and len(table) == 3


@pytest.mark.parametrize("seed", range(5))
def test_compact(seed):
    rng = random.Random(seed)
    bm = BlockManager(40, 4)
    tables, tokens = [], []
    for k in range(8):
        tok = [k] * rng.randint(1, 17)
        t, _ = bm.allocate(tok)
        tables.append(t)
        tokens.append(tok)
        bm.register_full_blocks(tok, t, len(tok))
    child, _ = bm.fork(tables[3], len(tokens[3]))
    for k in (1, 4, 6):
        bm.free_seq(tables[k])
    live = [t for t in tables if t] + [child]
    store = {b: ("block", b) for b in range(40)}
    before = [[store[b] for b in t] for t in live]
    cached = {h: store[b] for h, b in bm.block_of.items()}
    moves = bm.compact(live)
    for s, d in moves:
        store[d] = store[s]
    assert [[store[b] for b in t] for t in live] == before
    assert {h: store[b] for h, b in bm.block_of.items()} == cached
    used = {b for t in live for b in t} | set(bm.hash_of)
    assert used == set(range(len(used))) and sorted(bm.free) == list(range(len(used), 40))
    assert bm.num_free() == len(bm.free) + len(bm.evictable)
    again, _ = bm.allocate(tokens[1] + [99])  # the prefix cache still finds its blocks
    assert bm.stats.hits > 0 or len(tokens[1]) < 4
    for t in live + [again]:
        bm.free_seq(t)
    assert bm.num_free() == 40


def test_compact_wants_every_table():
    bm = BlockManager(8, 4)
    a, _ = bm.allocate([1] * 9)
    bm.allocate([2] * 3)
    with pytest.raises(ValueError):
        bm.compact([a])


# ------------------------------------------------------------------ engine
@pytest.mark.parametrize("prompt_len", [1, 4, 7, 13])
@pytest.mark.parametrize("blocks,seqs", [(64, 16), (9, 16), (64, 2)])
def test_samples_of_one_prompt(prompt_len, blocks, seqs):
    """n samples greedily: all equal the direct simulation, whether the others forked or had to wait."""
    eng, runner = _engine(blocks, max_num_seqs=max(seqs, 2))
    p = list(range(5, 5 + prompt_len))
    n = min(4, eng.sc.max_num_seqs)
    got = eng.generate([p, [3, 2, 1]], SamplingParams(max_tokens=9, n=n))
    assert got == [[reference(p, 9)] * n, [reference([3, 2, 1], 9)] * n]
    assert eng.blocks.num_free() == blocks
    if blocks == 64 and seqs == 16 and prompt_len % 4:
        assert len(runner.copied) == 3 + 3
        assert runner.prefill_rows == prompt_len + 3  # the prompts were computed once


def test_samples_without_page_copies():
    eng, _ = _engine(cls=KVRunner)
    assert eng.generate([[1, 2, 3]], SamplingParams(max_tokens=5, n=3)) == [[reference([1, 2, 3], 5)] * 3]


def test_fork_request_midway_and_compact():
    eng, runner = _engine(32)
    filler = [eng.add_request([k] * 11, SamplingParams(max_tokens=3 + 5 * (k % 2))) for k in range(4)]
    a = eng.add_request([5, 6, 7, 8, 9], SamplingParams(max_tokens=20))
    for _ in range(5):
        eng.step()
    seen = []
    b = eng.fork_request(a, SamplingParams(max_tokens=20, logit_bias={17: 1000.0}), on_token=lambda r, t: seen.append(t))
    c = eng.fork_request(a)
    common = list(next(r for r in eng.running if r.req_id == a).output)
    eng.step()
    used = 32 - len(eng.blocks.free)
    moved = eng.compact()
    assert moved > 0 and sorted(eng.blocks.free) == list(range(used, 32))
    _run(eng, [a, b, c] + filler)
    full = reference([5, 6, 7, 8, 9], 20)
    assert eng.finished[a].output == full and eng.finished[c].output == full
    assert eng.finished[b].output == common + [17] * (20 - len(common)) and seen == [17] * (20 - len(common))
    assert eng.blocks.num_free() == 32 and sorted(eng._counts_free) == list(range(eng._counts_rows))
    with pytest.raises(ValueError):
        eng.fork_request(a)


PARAMS = [dict(repetition_penalty=1.7), dict(frequency_penalty=0.9), dict(presence_penalty=1.1), dict(logit_bias={4: 3.0, 50: -20.0}),
          dict(allowed_token_ids=[3, 9, 27, 81]), dict(grammar=lambda out: [len(out), 40 + len(out)]),
          dict(grammar=lambda out: None if len(out) < 3 else [1, 2] if len(out) < 6 else []),
          dict(repetition_penalty=1.3, frequency_penalty=0.4, presence_penalty=0.2, logit_bias={8: 2.0}, allowed_token_ids=list(range(0, V, 2)))]


@pytest.mark.parametrize("blocks", [64, 14])
def test_adjusted_requests_in_one_batch(blocks):
    """Each request's own penalties and grammar, beside requests without any; with 14 blocks some are preempted, which
    takes their counts away and builds them again."""
    eng, _ = _engine(blocks, max_num_seqs=4)
    ps = [SamplingParams(max_tokens=12, **kw) for kw in PARAMS] + [SamplingParams(max_tokens=12)]
    prompts = [[k + 1, k + 2, k + 1, 30] for k in range(len(ps))]
    ids = [eng.add_request(p, sp) for p, sp in zip(prompts, ps)]
    _run(eng, ids)
    for i, p, sp in zip(ids, prompts, ps):
        want = _penalised(p, 12, sp)
        assert eng.finished[i].output == want, sp
        assert eng.finished[i].finish_reason == ("length" if len(want) == 12 else "stop")
    assert blocks == 64 or eng.stats["preemptions"] > 0
    assert eng.blocks.num_free() == blocks and sorted(eng._counts_free) == list(range(eng._counts_rows))


def test_refusals():
    eng, _ = _engine()
    for kw in (dict(repetition_penalty=0.0), dict(frequency_penalty=float("nan")), dict(presence_penalty=float("inf")),
               dict(logit_bias={V: 1.0}), dict(allowed_token_ids=[-1]), dict(allowed_token_ids=[]), dict(n=0), dict(n=10 ** 6)):
        with pytest.raises(ValueError):
            eng.add_request([1], SamplingParams(**kw))
    plain, _ = _engine(cls=KVRunner)
    for kw in (dict(repetition_penalty=1.1), dict(logit_bias={1: 1.0}), dict(allowed_token_ids=[1]), dict(grammar=lambda o: None)):
        with pytest.raises(ValueError, match="not supported"):
            plain.add_request([1], SamplingParams(**kw))
    with pytest.raises(ValueError):
        plain.compact()
    with pytest.raises(ValueError):
        eng.fork_request(123)


def test_validator_with_adjustments():
    v = InputValidator(100, adjust=True)
    v.check([1], {"presence_penalty": -2, "frequency_penalty": 1.5, "repetition_penalty": 1.2, "logit_bias": {"7": -100, "99": 3},
                  "allowed_token_ids": [1, 2]})
    v.check([1], {"presence_penalty": None, "logit_bias": None})
    for body in ({"presence_penalty": 2.5}, {"frequency_penalty": float("nan")}, {"frequency_penalty": True}, {"repetition_penalty": 0},
                 {"repetition_penalty": "2"}, {"logit_bias": [1]}, {"logit_bias": {"100": 1}}, {"logit_bias": {"-1": 1}},
                 {"logit_bias": {"a": 1}}, {"logit_bias": {"1": 101}}, {"logit_bias": {"1": None}}, {"logit_bias": {"²": 1}},
                 {"allowed_token_ids": []}, {"allowed_token_ids": [100]}, {"allowed_token_ids": [True]}, {"allowed_token_ids": 3}, {"n": 2}):
        with pytest.raises(ValidationError):
            v.check([1], body)


def _raises(out):
    raise RuntimeError("no such state")


@pytest.mark.parametrize("grammar,why", [(_raises, "RuntimeError: no such state"), (lambda out: [1, V], "token ids"), (lambda out: [-1], "token ids"),
                                         (lambda out: [0.5], "token ids"), (lambda out: 7, "TypeError")])
def test_a_failing_grammar_ends_its_own_request_only(grammar, why):
    eng, _ = _engine(max_num_seqs=8)
    late = SamplingParams(max_tokens=9, grammar=lambda out: None if len(out) < 4 else grammar(out), presence_penalty=0.5)
    ids = [eng.add_request([3, 4, 5], SamplingParams(max_tokens=9)), eng.add_request([3, 4, 5], SamplingParams(max_tokens=9, grammar=grammar)),
           eng.add_request([6, 7], late), eng.add_request([8, 9], SamplingParams(max_tokens=9, n=2, grammar=grammar))]
    _run(eng, ids)
    _run(eng, eng.finished[ids[3]].samples)
    assert eng.finished[ids[0]].output == reference([3, 4, 5], 9) and eng.finished[ids[0]].error is None
    for i, n in ((ids[1], 0), (ids[2], 4), (ids[3], 0), (eng.finished[ids[3]].samples[0], 0)):
        r = eng.finished[i]
        assert r.finish_reason == "error" and why in r.error and len(r.output) == n
    assert not eng.has_work() and eng.blocks.num_free() == 64 and sorted(eng._counts_free) == list(range(eng._counts_rows))


def test_grammars_may_return_any_collection_of_ids():
    """Lists, tuples, sets, ranges, generators and arrays alike; a set of fixed ids too."""
    import numpy as np
    want = {9, 27, 81}
    outs = []
    for kw in (dict(allowed_token_ids=want), dict(allowed_token_ids=np.array([9, 27, 81])), dict(grammar=lambda out: want), dict(grammar=lambda out: tuple(want)),
               dict(grammar=lambda out: (t for t in want)), dict(grammar=lambda out: np.array([9, 27, 81], dtype=np.int32)),
               dict(grammar=lambda out: range(9, 82), allowed_token_ids=want), dict(grammar=lambda out: None, allowed_token_ids=want)):
        eng, _ = _engine()
        i = eng.add_request([1, 2], SamplingParams(max_tokens=6, **kw))
        _run(eng, [i])
        outs.append(eng.finished[i].output)
    assert all(o == _penalised([1, 2], 6, SamplingParams(allowed_token_ids=[9, 27, 81])) for o in outs)


class PackingRunner(Runner):
    """Takes masks as the words that its pack_allowed makes, as the GPU runner does."""

    def pack_allowed(self, ids):
        import numpy as np
        assert isinstance(ids, np.ndarray) and ids.dtype == np.int64
        bits = np.zeros((V + 31) // 32 * 32, dtype=np.uint8)
        bits[ids] = 1
        return np.packbits(bits, bitorder="little").view(np.int32)

    def adjust_logits(self, logits, rows, penalties, biases, allowed):
        import numpy as np
        for a in allowed:
            assert a is None or (a.dtype == np.int32 and a.shape == ((V + 31) // 32,))
        ids = [None if a is None else np.flatnonzero(np.unpackbits(a.view(np.uint8), bitorder="little")) for a in allowed]
        return super().adjust_logits(logits, rows, penalties, biases, ids)


def test_grammar_arrays_are_ids_not_mask_words():
    import numpy as np
    for words in (np.array([5, 6, 7, 8]), np.array([5, 6, 7, 8], dtype=np.int32), {5, 6, 7, 8}):
        eng, _ = _engine(cls=PackingRunner)
        i = eng.add_request([1, 2], SamplingParams(max_tokens=4, grammar=lambda out: words[len(out):len(out) + 1] if isinstance(words, np.ndarray) else words))
        _run(eng, [i])
        assert set(eng.finished[i].output) <= {5, 6, 7, 8} and eng.finished[i].finish_reason == "length"


def test_on_finish_is_called_once_however_a_request_ends():
    """With a last token, without any, aborted while it waits and while it runs, and for each of several samples."""
    eng, _ = _engine(max_num_seqs=4)
    ended = []
    add = lambda **kw: eng.add_request([3, 4, 5], SamplingParams(max_tokens=6, **kw), on_finish=lambda r: ended.append((r.req_id, r.finish_reason, len(r.output))))  # noqa: E731
    a, b, c, d = add(), add(grammar=lambda out: [] if len(out) == 2 else None), add(grammar=_raises), add(n=2)
    e, f = add(), add()
    eng.abort_request(f)
    eng.step()
    g = eng.fork_request(a, on_finish=lambda r: ended.append((r.req_id, r.finish_reason, len(r.output))))
    eng.abort_request(a)
    _run(eng, [a, b, c, d, e, f, g])
    _run(eng, eng.finished[d].samples)
    assert sorted(ended) == sorted([(a, "abort", 1), (b, "stop", 2), (c, "error", 0), (d, "length", 6), (eng.finished[d].samples[0], "length", 6),
                                    (e, "length", 6), (f, "abort", 0), (g, "length", 6)])
    assert all(r.finished for r in eng.finished.values()) and eng.blocks.num_free() == 64


def test_seeded_samples_and_forks_repeat():
    """Every sample and fork of a seeded request draws with a seed of its own, the same one whatever else the engine served before."""
    def seeds(busy):
        eng, _ = _engine(max_num_seqs=8)
        for k in range(busy):
            _run(eng, [eng.add_request([k + 1], SamplingParams(max_tokens=2))])
        i = eng.add_request([1, 2, 3], SamplingParams(max_tokens=6, temperature=1.0, seed=7, n=3))
        eng.step()
        kids = next(r for r in eng.running if r.req_id == i).samples + [eng.fork_request(i), eng.fork_request(i)]
        _run(eng, [i] + kids)
        return [eng.finished[k].params.seed for k in [i] + kids]
    first = seeds(0)
    assert seeds(3) == first and first[0] == 7 and len(set(first)) == 5 and all(0 <= s < 2 ** 63 for s in first)


@pytest.mark.parametrize("kw", [dict(temperature=1.0, top_p=0.9), dict(temperature=1.0, seed=4), dict(logit_bias={1: 1.0})])
def test_fork_request_refuses_what_add_request_refuses(kw):
    """A runner without top_p, seeds and logits changes: refused at the fork, not inside a step; the first request goes on."""
    eng, _ = _engine(cls=KVRunner)
    i = eng.add_request([1, 2, 3], SamplingParams(max_tokens=6))
    eng.step()
    for add in (lambda p: eng.add_request([1], p), lambda p: eng.fork_request(i, p)):
        with pytest.raises(ValueError, match="not supported"):
            add(SamplingParams(max_tokens=6, **kw))
    _run(eng, [i])
    assert eng.finished[i].output == reference([1, 2, 3], 6) and not eng.has_work()


def test_fork_request_keeps_to_max_tokens():
    """max_tokens bounds a fork's whole output: a fork that has it already is refused."""
    eng, _ = _engine()
    i = eng.add_request([1, 2, 3], SamplingParams(max_tokens=9))
    for _ in range(4):
        eng.step()
    have = len(next(r for r in eng.running if r.req_id == i).output)
    with pytest.raises(ValueError, match="max_tokens"):
        eng.fork_request(i, SamplingParams(max_tokens=have))
    j = eng.fork_request(i, SamplingParams(max_tokens=have + 1))
    _run(eng, [i, j])
    assert eng.finished[j].output == reference([1, 2, 3], have + 1) and eng.finished[i].output == reference([1, 2, 3], 9)


def test_a_fork_that_waits_keeps_its_priority():
    eng, _ = _engine(max_num_seqs=2)
    a = eng.add_request([1, 2, 3], SamplingParams(max_tokens=30), priority=1)
    b = eng.add_request([4, 5, 6], SamplingParams(max_tokens=30), priority=1)
    for _ in range(3):
        eng.step()
    queued = {p: eng.add_request([7, 8], SamplingParams(max_tokens=3), priority=p) for p in (0, 1, 2)}
    c = eng.fork_request(a)
    assert [r.req_id for r in eng.waiting] == [queued[0], c, queued[1], queued[2]]
    _run(eng, [a, b, c] + list(queued.values()))
    assert eng.finished[c].output == reference([1, 2, 3], 30)


def test_times_of_samples_and_forks():
    """Queue time, time to first token and token times of each are its own: none negative, none from before it arrived."""
    eng, _ = _engine(max_num_seqs=3)
    now = [0.0]
    eng.clock = lambda: now[0]
    i = eng.add_request([1, 2, 3], SamplingParams(max_tokens=6, n=2))
    now[0] = 1.0
    eng.step()
    now[0] = 2.0
    eng.step()
    now[0] = 3.0
    kids = next(r for r in eng.running if r.req_id == i).samples + [eng.fork_request(i), eng.fork_request(i)]  # the last one waits
    while any(k not in eng.finished for k in [i] + kids):
        now[0] += 1.0
        eng.step()
    for k, arrived, own in ((i, 0.0, 6), (kids[0], 0.0, 6), (kids[1], 3.0, 4), (kids[2], 3.0, 4)):
        r = eng.finished[k]
        assert r.output == reference([1, 2, 3], 6) and r.arrival == arrived and len(r.token_times) == own
        assert r.arrival <= r.scheduled_time <= r.first_token_time == r.token_times[0] and r.token_times == sorted(r.token_times)
    assert eng.finished[kids[0]].first_token_time == eng.finished[i].first_token_time == 1.0


REFUSED = [{"repetition_penalty": 1.1}, {"logit_bias": {"7": 5}}, {"allowed_token_ids": [1, 2]}, {"allowed_token_ids": []}, {"logit_bias": [1]}]
NEUTRAL = [{"repetition_penalty": 1.0}, {"repetition_penalty": None, "logit_bias": {}, "allowed_token_ids": None}, {"logit_bias": None}]


def test_validator_without_adjustments_refuses_them():
    v = InputValidator(100)
    for body in NEUTRAL:
        v.check([1], body)
    for body in REFUSED + [{"presence_penalty": 0.5}, {"frequency_penalty": -0.5}]:
        with pytest.raises(ValidationError, match="not supported"):
            v.check([1], body)


@pytest.mark.parametrize("own_validator", [False, True])
def test_server_without_adjustments_refuses_them(own_validator):
    """Over HTTP, chat and the WebSocket, with the server's validator and with one of the caller's that knows nothing of these fields."""
    from test_server_cpu import _run as serve

    class Lenient:
        def check(self, ids, body):
            pass

    async def go(client):
        for body in REFUSED:
            r = await client.post("/v1/completions", json={"prompt": "ab", "max_tokens": 2, **body})
            assert r.status == 400 and "not supported" in (await r.json())["error"]["message"]
            r = await client.post("/v1/chat/completions", json={"messages": [{"role": "user", "content": "a"}], "max_tokens": 2, **body})
            assert r.status == 400
        for body in NEUTRAL:
            r = await client.post("/v1/completions", json={"prompt": "ab", "max_tokens": 2, **body})
            assert r.status == 200 and len((await r.json())["token_ids"]) == 2
        ws = await client.ws_connect("/v1/ws")
        await ws.send_json({"prompt": "ab", "max_tokens": 2, "allowed_token_ids": [5]})
        assert "not supported" in (await ws.receive_json())["error"]["message"]
        await ws.send_json({"prompt": "ab", "max_tokens": 1})
        assert "token" in await ws.receive_json()
        await ws.close()
    serve(go, **({"validator": Lenient()} if own_validator else {}))


def test_values_outside_fp32_are_refused():
    """What fp32 turns into 0, infinity or NaN would spoil a row of logits; -inf bans a token."""
    eng, _ = _engine()
    for kw in (dict(repetition_penalty=1e-50), dict(repetition_penalty=1e39), dict(repetition_penalty=2.0 ** -127), dict(repetition_penalty=float("nan")),
               dict(frequency_penalty=1e39), dict(presence_penalty=-1e39), dict(logit_bias={3: float("nan")}), dict(logit_bias={3: float("inf")}),
               dict(logit_bias={3: 1e39}), dict(logit_bias={3: -float("inf"), 4: -float("inf")}, allowed_token_ids=[4, 3, 4])):
        with pytest.raises(ValueError):
            eng.add_request([1], SamplingParams(**kw))
    ban = -float("inf")
    for kw, want in ((dict(logit_bias={9: ban}, allowed_token_ids=[9, 27]), [27] * 4), (dict(logit_bias={9: ban, 27: ban}, grammar=lambda out: [9, 27]), []),
                     (dict(logit_bias={9: ban}, grammar=lambda out: [9, 27] if len(out) < 2 else [9]), [27, 27])):
        i = eng.add_request([1, 2], SamplingParams(max_tokens=4, **kw))
        _run(eng, [i])
        assert eng.finished[i].output == want and eng.finished[i].finish_reason == ("length" if len(want) == 4 else "stop")


def test_chunks_that_attend_to_the_pages_are_bounded_by_query_rows():
    """Heads count as tokens do: the longest such chunk shrinks with them (128 tokens of 64 heads were slower than a copy)."""
    from types import SimpleNamespace
    from lora_kernel_b200.serve.model_runner import ModelRunner
    longest = lambda h, dh, rows=ModelRunner.PAGE_ATTN_ROWS: ModelRunner.page_attn_tokens.fget(  # noqa: E731
        SimpleNamespace(cfg=SimpleNamespace(num_heads=h, head_dim=dh), PAGE_ATTN_ROWS=rows))
    assert longest(32, 128) == 128 and longest(64, 128) == 64 and longest(8, 128) == 512
    assert longest(32, 64) == 192 and longest(64, 64) == 96 and longest(8, 64) == 768
    assert longest(28, 128) == 146 and longest(32, 128, 0) == 0


# ------------------------------------------------------------------ the oracles themselves
def test_page_oracle_properties():
    import paged_oracle as O
    for dtype, q in O.QMAX.items():
        for amax in (0.0, 1e-40, 1.0, q, q * 1.001, q * 2.0 ** 20, 3e38):
            s = O.page_scale(amax, q)
            assert amax <= s * q and (s == 2.0 ** -126 or amax > s / 2 * q)
    x = torch.randn(1000, dtype=torch.float64) * 100
    codes = O.encode(x, torch.float8_e4m3fn)
    assert torch.equal(codes.float().to(torch.float8_e4m3fn).double(), codes)  # they are e4m3 values
    assert torch.equal(codes, x.float().to(torch.float8_e4m3fn).double())      # and the nearest ones
    q, k, v = torch.randn(3, 4, 8).double(), torch.randn(7, 2, 8).double(), torch.randn(7, 2, 8).double()
    out, mag = O.attention(q, k, v, 7, 3)
    assert (mag >= out.abs()).all()
    alone, _ = O.attention(q[:1], k[:5], v[:5], 5, 1)
    assert torch.allclose(out[0], alone[0])
    assert not O.attention(q, k[:1], v[:1], 1, 3)[0][:2].any()


def test_ops_refuse_cpu_tensors():
    from lora_kernel_b200.ops import logits as LG
    from lora_kernel_b200.ops import paged as PG
    z = torch.zeros(1, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        PG.page_attention(z, z, z, z, z, i, i, 16, 1, 1, 64)
    with pytest.raises(RuntimeError):
        PG.page_append(z, 1, 1, 64, i, z, z, z, z, 16)
    with pytest.raises(RuntimeError):
        PG.copy_pages([z], [(0, 1)], 1)
    with pytest.raises(RuntimeError):
        LG.adjust_logits(z)
