"""Serving over the page-scaled cache on the GPU: the engine's logits, CUDA-graph decode, forks, compaction, penalties
and grammars on the path that a user takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
dev = "cuda"


def _engine(kv, graphs=False, prefix=True, **kw):
    from lora_kernel_b200.config import ServeConfig, TransformerConfig
    from lora_kernel_b200.models.params import FlatParams
    from lora_kernel_b200.serve.engine import LLMEngine
    cfg = TransformerConfig(hidden_dim=256, num_heads=8, num_kv_heads=2, head_dim=64, ff_dim=512, vocab_size=1000,
                            num_layers=3, max_seq_len=1024)
    params = FlatParams(cfg, dev)
    params.init_(0, 0.05)
    sc = ServeConfig(num_kv_blocks=128, block_size=16, max_num_batched_tokens=512, max_model_len=1024, cuda_graphs=graphs,
                     enable_prefix_caching=prefix, **kw)
    return cfg, params, LLMEngine(cfg, params, sc, kv_dtype=kv)


def _tokens(n, seed, vocab=1000):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _status_ok():
    from lora_kernel_b200._ext import check_status
    check_status()


@pytest.mark.parametrize("kv", ["fp8_page", "int8_page"])
def test_logits_match_full_forward(kv):
    """Prefill in two chunks, a short chunk over the pages, decode steps, against the training model's forward
    (the cache rounds to 2^-4 of an element in fp8, 2^-7 of the page's largest in int8: the same bound as for the
    caches with a scale per token)."""
    from lora_kernel_b200.models.llama import LlamaModel
    from lora_kernel_b200.serve.model_runner import PrefillItem
    cfg, params, eng = _engine(kv)
    model = LlamaModel(cfg, dev, params=params, with_grads=False)
    seq = _tokens(300, 4)
    full = model.forward(torch.tensor([seq], device=dev))[0].float()
    r = eng.runner
    table, _ = eng.blocks.allocate(seq)
    slots = eng.blocks.slots_for(table, 0, 300)
    r.prefill([PrefillItem(0, seq[:120], 0, slots, False)])
    got = {}
    _, lg = r.prefill([PrefillItem(0, seq[120:200], 120, slots, True)])
    got[199] = lg[0]
    _, lg = r.prefill([PrefillItem(0, seq[200:207], 200, slots, True, True)])  # 7 rows: attends to the pages
    for k in range(7):
        got[200 + k] = lg[k]
    for p in range(207, 211):
        got[p] = r.decode([seq[p]], [p], [slots[p]], [table])[0]
    for p, row in got.items():
        rel = ((row.float() - full[p]).norm() / full[p].norm()).item()
        assert rel < 0.2, (p, rel)
    _status_ok()


@pytest.mark.parametrize("kv", ["fp8_page", "int8_page"])
def test_short_chunks_agree_with_the_gathered_path(kv):
    """The same chunk over the pages and over their bf16 copy: both attend to the same cached values, so only the
    kernels' roundings are between them (bf16 outputs, 2^-9 an attention)."""
    from lora_kernel_b200.serve.model_runner import PrefillItem
    cfg, params, eng = _engine(kv)
    r, seq = eng.runner, _tokens(180, 5)
    table, _ = eng.blocks.allocate(seq)
    slots = eng.blocks.slots_for(table, 0, 180)
    out = []
    for rows in (type(r).PAGE_ATTN_ROWS, 0):
        r.PAGE_ATTN_ROWS = rows
        r.prefill([PrefillItem(0, seq[:171], 0, slots, False)])
        out.append(r.prefill([PrefillItem(0, seq[171:], 171, slots, True, True)])[1].float())
    assert out[0].shape == (9, cfg.vocab_size)
    assert ((out[0] - out[1]).norm() / out[1].norm()).item() < 2e-2


@pytest.mark.parametrize("kv", ["fp8_page", "int8_page"])
def test_graph_decode_matches_eager(kv):
    from lora_kernel_b200.serve.model_runner import PrefillItem
    cfg, params, eng = _engine(kv)
    r = eng.runner
    seqs = [_tokens(n, n) for n in (30, 75, 140)]
    tables = []
    for k, s in enumerate(seqs):
        table, _ = eng.blocks.allocate(s)
        r.prefill([PrefillItem(k, s[:-1], 0, eng.blocks.slots_for(table, 0, len(s) - 1), False)])
        tables.append(table)
    toks, pos = [s[-1] for s in seqs], [len(s) - 1 for s in seqs]
    sl = [eng.blocks.append_slot(t, p) for t, p in zip(tables, pos)]
    eager = r.decode(toks, pos, sl, tables).float().clone()
    r.enable_graphs(capture=False)
    for _ in range(2):  # the first call captures (3 rows in a bucket of 4), the second replays
        got = r.decode(toks, pos, sl, tables).float()
        assert ((got - eager).norm() / eager.norm()).item() < 1e-2
    _status_ok()


@pytest.mark.parametrize("kv", ["bf16", "fp8", "int8", "fp8_page", "int8_page"])
def test_fork_and_compact_keep_the_cache(kv):
    """A fork reads what its parent reads, and compaction changes nothing that is read: logits to the bit."""
    from lora_kernel_b200.serve.model_runner import PrefillItem
    cfg, params, eng = _engine(kv, prefix=False)
    r, bm = eng.runner, eng.blocks
    a, b = _tokens(53, 1), _tokens(40, 2)
    ta, _ = bm.allocate(a)
    gone, _ = bm.allocate(_tokens(100, 3))
    tb, _ = bm.allocate(b)
    r.prefill([PrefillItem(0, a, 0, bm.slots_for(ta, 0, 53), False), PrefillItem(1, b, 0, bm.slots_for(tb, 0, 40), False)])
    child, copies = bm.fork(ta, 53)
    assert len(copies) == 1
    r.copy_pages(copies)

    def decode():
        tables = [ta, tb, child]
        slots = [bm.slots_for(t, p, p + 1)[0] for t, p in zip(tables, (53, 40, 53))]
        return r.decode([7, 8, 7], [53, 40, 53], slots, tables).clone()

    bm.append_slot(tb, 40)
    first = decode()
    assert torch.equal(first[0], first[2])
    bm.free_seq(gone)
    moves = bm.compact([ta, tb, child])
    assert moves
    r.copy_pages(moves)
    assert torch.equal(decode(), first)
    _status_ok()


@pytest.mark.parametrize("graphs", [False, True])
def test_samples_with_penalties_and_grammars(graphs):
    """Several samples of one prompt, penalties, biases and grammars in one batch, through LLMEngine.generate."""
    from lora_kernel_b200.serve.engine import SamplingParams
    cfg, params, eng = _engine("fp8_page", graphs, max_num_seqs=16)
    prompt = _tokens(37, 9)
    outs = eng.generate([prompt], SamplingParams(max_tokens=12, n=5, temperature=1.0, seed=3))[0]
    assert len(outs) == 5 and all(len(o) == 12 for o in outs) and len({tuple(o) for o in outs}) == 5
    greedy = eng.generate([prompt], SamplingParams(max_tokens=12, n=3))[0]
    assert greedy[0][0] == greedy[1][0] == greedy[2][0]
    plan = [SamplingParams(max_tokens=20, allowed_token_ids=[5, 700, 999]),
            SamplingParams(max_tokens=20, presence_penalty=1000.0),
            SamplingParams(max_tokens=20, logit_bias={123: 10000.0}),
            SamplingParams(max_tokens=20, grammar=lambda out: [len(out) * 3 % 1000]),
            SamplingParams(max_tokens=20),
            SamplingParams(max_tokens=20, temperature=1.0, seed=1, frequency_penalty=1000.0, allowed_token_ids=list(range(40, 60)))]
    ids = [eng.add_request(prompt, p) for p in plan]
    while any(i not in eng.finished for i in ids):
        eng.step()
    out = [eng.finished[i].output for i in ids]
    assert set(out[0]) <= {5, 700, 999}
    assert len(set(out[1])) == 20
    assert out[2] == [123] * 20
    assert out[3] == [k * 3 for k in range(20)]
    assert out[4][0] == greedy[0][0]
    assert sorted(out[5]) == list(range(40, 60))
    assert eng.blocks.num_free() == eng.blocks.num_blocks and sorted(eng._counts_free) == list(range(eng._counts_rows))
    _status_ok()


def test_speculative_decoding_over_pages():
    """Draft and target over page-scaled caches; with the target as its own draft nearly everything is accepted (near
    ties aside: a chunk of rows and a decode step round differently)."""
    from lora_kernel_b200.serve.speculative import RunnerScorer, SpeculativeDecoder
    cfg, params, eng = _engine("fp8_page")
    _, _, other = _engine("fp8_page")
    dec = SpeculativeDecoder(RunnerScorer(eng.runner), RunnerScorer(other.runner), k=4)
    out = dec.generate(_tokens(50, 11), 40)
    assert len(out) == 40 and dec.stats.acceptance_rate > 0.5
    with pytest.raises(ValueError):
        RunnerScorer(eng.runner, base_slot=8)
    _status_ok()


@pytest.mark.parametrize("kv", ["fp8_page", "int8_page"])
def test_rejected_rows_leave_no_trace_in_a_page(kv):
    """Rows dropped by truncate do not raise the scale of the page that the kept ones end in: scales and logits are those
    of a sequence that never had them.  (A page's largest value may differ by the roundings of another chunk size, some
    percent after three layers: scales whose bound is nearer than that are left out.)"""
    from lora_kernel_b200.serve.speculative import RunnerScorer
    _, _, ea = _engine(kv)
    _, _, eb = _engine(kv)
    a, b = RunnerScorer(ea.runner), RunnerScorer(eb.runner)
    drafts = _tokens(1, 12) + [999] * 12
    for s in (a, b):
        s.runner.W["embed"][999] = s.runner.W["layers.0.wqkv"][8 * 64]  # a token with a large key (layer 0, head 0, dim 0)
        s.extend(_tokens(50, 11, 999), False)
    a.extend(drafts, True)
    raised = float(ea.runner.k_scale[0, 3, 0])
    a.truncate(51)
    b.extend(drafts[:1], True)
    la, lb = a.extend(_tokens(3, 13, 999), True), b.extend(_tokens(3, 13, 999), True)
    assert la.shape == lb.shape == (3, 1000) and a.length == b.length == 54
    q = {"fp8_page": 448.0, "int8_page": 127.0}[kv]
    assert raised >= 2 * float(eb.runner.k_scale[0, 3, 0]) == 2 * float(ea.runner.k_scale[0, 3, 0])
    for sa, sb, codes in ((ea.runner.k_scale, eb.runner.k_scale, eb.runner.k_cache), (ea.runner.v_scale, eb.runner.v_scale, eb.runner.v_cache)):
        assert torch.equal(sa[:, :3], sb[:, :3])
        filled = codes[:, 48:54].float().abs().amax(dim=(1, 3)) / q  # of the page's largest value, 1/2 to 1
        clear = (filled > 0.54) & (filled < 0.95)
        assert torch.equal(sa[:, 3][clear], sb[:, 3][clear])
    assert ((la - lb).norm() / lb.norm()).item() < 5e-2
    _status_ok()
