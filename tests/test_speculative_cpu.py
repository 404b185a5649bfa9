"""Speculative decoding on CPU with table (bigram) models: greedy output is the
target's own greedy decode, and speculative sampling draws from the target
distribution."""
import pytest
import torch

from lora_kernel_b200.serve.speculative import Scorer, SpeculativeDecoder, greedy_reference


class Bigram(Scorer):
    """Next-token logits depend on the current token only: logits[t] = table[t]."""

    def __init__(self, table: torch.Tensor):
        self.table = table
        self._len = 0
        self.calls = 0

    @property
    def length(self):
        return self._len

    def extend(self, tokens, all_logits):
        self.calls += 1
        self._len += len(tokens)
        rows = self.table[torch.tensor(tokens)]
        return rows if all_logits else rows[-1:]

    def truncate(self, length):
        self._len = min(self._len, length)


def _table(V, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(V, V, generator=g) * scale


@pytest.mark.parametrize("k", [1, 3, 5])
def test_greedy_speculative_equals_target_greedy(k):
    V = 50
    target, draft = Bigram(_table(V, 1)), Bigram(_table(V, 2))
    prompt = [3, 17, 9]
    ref = greedy_reference(Bigram(target.table), prompt, 40)
    sd = SpeculativeDecoder(target, draft, k=k)
    assert sd.generate(prompt, 40) == ref
    assert sd.stats.emitted == 40
    # fewer target forwards than tokens unless every proposal is rejected
    assert sd.stats.target_forwards <= 40


def test_identical_draft_accepts_everything():
    V = 30
    t = _table(V, 4)
    sd = SpeculativeDecoder(Bigram(t), Bigram(t.clone()), k=4)
    out = sd.generate([1, 2], 20)
    assert out == greedy_reference(Bigram(t), [1, 2], 20)
    assert sd.stats.acceptance_rate == 1.0
    assert sd.stats.tokens_per_target_forward == pytest.approx(5.0)


def test_partially_matching_draft():
    # the draft agrees with the target on half of the vocabulary
    V = 40
    t = _table(V, 5)
    d = _table(V, 6)
    d[: V // 2] = t[: V // 2]
    sd = SpeculativeDecoder(Bigram(t), Bigram(d), k=4)
    assert sd.generate([7], 60) == greedy_reference(Bigram(t), [7], 60)
    assert 0.0 < sd.stats.acceptance_rate < 1.0


def test_eos_and_length_limits():
    V = 20
    t = _table(V, 7)
    ref = greedy_reference(Bigram(t), [0], 30)
    eos = ref[5]
    first = ref.index(eos)
    sd = SpeculativeDecoder(Bigram(t), Bigram(_table(V, 8)), k=3, eos_id=eos)
    assert sd.generate([0], 30) == ref[:first + 1]
    sd2 = SpeculativeDecoder(Bigram(t), Bigram(_table(V, 8)), k=4)
    assert len(sd2.generate([0], 7)) == 7


def test_speculative_sampling_matches_target_distribution():
    V, runs = 5, 6000
    t, d = _table(V, 11, 1.0), _table(V, 12, 1.0)
    temp = 0.8
    p = torch.softmax(t / temp, dim=-1)
    # distribution of the 2nd generated token after prompt [2]: sum_a p(a|2) p(b|a)
    want = p[2] @ p
    counts = torch.zeros(V)
    for s in range(runs):
        sd = SpeculativeDecoder(Bigram(t), Bigram(d), k=3, temperature=temp, seed=s)
        out = sd.generate([2], 2)
        counts[out[1]] += 1
    e = want * runs
    chi2 = float(((counts - e) ** 2 / e).sum())
    assert chi2 < 25.0, (counts / runs, want)  # 4 dof: p ~ 5e-5


class PageRunner:
    """Keeps what an append does to a page's scale: offset 0 starts the page afresh, later rows can only raise it."""

    def __init__(self, page_scaled, block_size=8, num_blocks=8):
        self.page_scaled, self.block_size, self.num_blocks, self.max_model_len = page_scaled, block_size, num_blocks, block_size * num_blocks
        self.slot, self.scale, self.rows = {}, {}, 0

    def prefill(self, items):
        (it,) = items
        assert it.want_logits and len(it.slots) == it.start + len(it.tokens)
        for t, s in zip(it.tokens, it.slots[it.start:]):
            page, off = divmod(s, self.block_size)
            self.scale[page] = t if off == 0 else max(self.scale[page], t)
            self.slot[s] = t
        self.rows += len(it.tokens)
        seen = [self.slot[s] for s in it.slots]
        n = len(it.tokens) if it.all_logits else 1
        return [it.seq_id], torch.tensor([[float(sum(seen[:len(seen) - n + k + 1])), float(len(seen) - n + k)] for k in range(n)])


@pytest.mark.parametrize("page_scaled", [True, False])
@pytest.mark.parametrize("prompt,drafts,keep", [(5, 2, 1), (8, 3, 0), (13, 12, 1), (13, 12, 3), (20, 5, 4), (20, 5, 5), (3, 20, 14), (1, 1, 0)])
def test_dropped_rows_leave_no_trace_in_a_page(page_scaled, prompt, drafts, keep):
    """After truncate and the next rows, tokens, page scales and logits are those of a sequence that never had the dropped rows."""
    from lora_kernel_b200.serve.speculative import RunnerScorer
    a, b = PageRunner(page_scaled), PageRunner(page_scaled)
    sa, sb = RunnerScorer(a, base_slot=16, max_len=48), RunnerScorer(b, base_slot=16, max_len=48)
    d = list(range(100, 100 + drafts))
    for s in (sa, sb):
        s.extend(list(range(1, prompt + 1)), False)
    sa.extend(d, True)
    sa.truncate(prompt + keep)
    assert sa.length == prompt + keep
    if keep:
        sb.extend(d[:keep], True)
    for nxt, every in (([3, 4, 5], True), ([6], False)):
        la, lb = sa.extend(nxt, every), sb.extend(nxt, every)
        assert torch.equal(la, lb) and sa.length == sb.length
    pages = {s // 8 for s in range(16, 16 + sa.length)}
    assert {p: a.scale[p] for p in pages} == {p: b.scale[p] for p in pages} or not page_scaled
    assert all(a.slot[s] == b.slot[s] for s in range(16, 16 + sa.length))
    if not page_scaled:
        assert a.rows == prompt + drafts + 4  # nothing is computed twice
    sa.truncate(0)
    assert sa.length == 0 and torch.equal(sa.extend([9, 9], True), torch.tensor([[9.0, 0.0], [18.0, 1.0]]))
