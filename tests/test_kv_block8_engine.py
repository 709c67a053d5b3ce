"""Serving over the block-scaled 8-bit KV cache (kv_cache_dtype int8 / fp8_block) and eviction by attention weight
(kv_eviction_policy attention): tokens against the fp32 decoder, the sequence tables, the refusals."""
import pytest
import torch

from gollek_b200.config import EngineConfig, preset
from gollek_b200.engine.engine import LLMEngine
from gollek_b200.engine.sequence import SamplingParams
from gollek_b200.models.reference import ReferenceDecoder, init_random_weights
from gollek_b200.native import host_ext
from gollek_b200.utils.tokenizer import ByteTokenizer


def engine(cfg, weights, device="cpu", num_blocks=128, **kw):
    base = dict(device=device, max_num_seqs=4, max_num_batched_tokens=512, max_model_len=512, kv_cache_dtype="int8")
    if device == "cpu":
        base.update(dtype="float32", use_cuda_graphs=False, async_scheduling=False)
    else:
        base.update(cuda_graph_batch_sizes=(1, 2, 4))
    base.update(kw)
    return LLMEngine(EngineConfig(**base), model_cfg=cfg, weights=weights.__getitem__, num_blocks=num_blocks,
                     tokenizer=ByteTokenizer(cfg.vocab_size, cfg.eos_token_id))


def gaps(cfg, weights, prompt, tokens, key_mask=None):
    """How far below the fp32 decoder's best logit each produced token lies, in standard deviations of its logits."""
    s = prompt + list(tokens)
    logits = ReferenceDecoder(cfg, weights).forward(torch.tensor(s), key_mask)[len(prompt) - 1: len(s) - 1]
    return (logits.max(-1).values - logits[torch.arange(len(tokens)), torch.tensor(tokens)]) / logits.std(-1)


# int8 codes keep 7 bits below a block's largest value (half a step 2^-7 .. 2^-8 of it), e4m3 half a step 2^-4 of each
# value: the latter is what the per-token fp8 cache keeps, for which 0.25 of a standard deviation is the bound in use
@pytest.mark.parametrize("kind", ["int8", "fp8_block"])
@pytest.mark.parametrize("block_size", [16, 32])
def test_engine_tokens_cpu(tiny_cfg, tiny_weights, kind, block_size):
    eng = engine(tiny_cfg, tiny_weights, kv_cache_dtype=kind, block_size=block_size)
    assert eng.kv_cache.dtype == (torch.int8 if kind == "int8" else torch.uint8)
    assert tuple(eng.model.kv_scales.shape) == tuple(eng.kv_cache.shape[:4]) and eng.model.kv_mass is None
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(3, 250, (n,), generator=g).tolist() for n in (90, 17, 33)]
    prompts.append(prompts[0][:64] + [7, 8, 9])                  # shares blocks with the first one's prefix
    for _ in range(2):                                            # the second time over cached prefixes
        outs = eng.generate(prompts, SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True))
        for p, o in zip(prompts, outs):
            assert float(gaps(tiny_cfg, tiny_weights, p, o.output_token_ids).max()) < 0.25
    assert eng.kv.prefix_hits > 0


def test_compact_tables():
    h = host_ext()
    pool = h.BlockPool(32, 4)
    t = h.SeqTables(pool)
    t.add(7)
    assert t.ensure_capacity(7, 18)                               # 5 blocks of 4
    blocks = t.blocks(7)
    assert t.compact(7, 18, 9) == 2 and t.dropped(7) == 9 and t.blocks(7) == blocks[:3]
    assert pool.num_free() == 32 - 3
    for bad in ((18, 9), (12, 0), (9, 10)):                       # more tokens than blocks hold, none kept, more than all
        with pytest.raises(Exception):
            t.compact(7, *bad)
    pos, slots, bt = (torch.zeros(*s, dtype=torch.int32) for s in ((4,), (4,), (1, 8)))
    lens, qs = torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    t.build_batch(torch.tensor([7]), torch.tensor([18], dtype=torch.int32), torch.tensor([1], dtype=torch.int32), pos,
                  slots, bt, lens, qs)
    assert int(pos[0]) == 18 and int(lens[0]) == 10 and int(slots[0]) == blocks[2] * 4 + 1
    assert t.blocks_needed(7, 21) == 0 and t.blocks_needed(7, 22) == 1


def evicted_run(cfg, weights, device, **kw):
    """Prefill, give every head the same weights, evict, decode on; returns what the masked decoder needs."""
    eng = engine(cfg, weights, device=device, kv_eviction=True, kv_eviction_policy="attention",
                 kv_eviction_threshold=1.1, kv_retention_target=0.5, kv_eviction_min_blocks=4, **kw)
    assert not eng.cfg.enable_prefix_caching
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(3, 250, (203,), generator=g).tolist()
    eng.add_request("r", prompt, SamplingParams(temperature=0.0, max_tokens=10, ignore_eos=True))
    eng.step()
    seq = next(iter(eng.seqs.values()))
    while seq.num_computed_tokens < len(prompt):
        eng.step()
    m = eng.model
    # the prompt chunk's last query has weighed every token: one softmax per query head
    total = float(m.kv_mass.double().sum())
    tokens = seq.num_computed_tokens - eng.kv.dropped_tokens(seq)
    blocks = torch.tensor(eng.kv.tables.blocks(seq.seq_id)).to(m.kv_mass.device)
    w = torch.rand(tokens, generator=g).to(m.kv_mass.device)
    at = torch.arange(tokens, device=w.device)
    m.kv_mass[:, blocks[at // 16], :, at % 16] = w[:, None, None].expand(-1, m.kv_mass.shape[0], m.Hk)
    nb = len(blocks)
    freed = eng.evictor.run(eng, force=True)
    keep = -(-nb // 2) * 16
    assert freed == nb - keep // 16 and eng.kv.dropped_tokens(seq) == tokens - keep
    a, r = 16, -(-tokens // 5)
    mid = w[a:tokens - r].cpu().sort(descending=True, stable=True).indices[: keep - a - r] + a
    gone = sorted(set(range(a, tokens - r)) - set(mid.tolist()))
    out = None
    while eng.has_unfinished():
        for o in eng.step():
            if o.finished:
                out = o
    return eng, prompt, list(out.output_token_ids), gone, tokens, total


def check_evicted(cfg, weights, prompt, toks, gone, tokens):
    n = len(prompt) + len(toks)
    mask = torch.ones(n, n, dtype=torch.bool)
    mask[tokens:, gone] = False                                   # queries after the eviction do not see them
    assert float(gaps(cfg, weights, prompt, toks, mask).max()) < 0.25


def test_decode_after_eviction_matches_masked_decoder(tiny_cfg, tiny_weights):
    eng, prompt, toks, gone, tokens, total = evicted_run(tiny_cfg, tiny_weights, "cpu")
    check_evicted(tiny_cfg, tiny_weights, prompt, toks, gone, tokens)
    assert abs(total - tiny_cfg.num_hidden_layers * tiny_cfg.num_attention_heads) < 1e-3
    assert eng.evictor.stats.sequences == 1 and eng.kv.num_free_blocks() == eng.num_blocks


def test_pressure_evicts_instead_of_preempting(tiny_cfg, tiny_weights):
    eng = engine(tiny_cfg, tiny_weights, num_blocks=40, kv_eviction=True, kv_eviction_policy="attention",
                 kv_eviction_threshold=0.8, kv_retention_target=0.6, kv_eviction_min_blocks=4)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(3, 250, (n,), generator=g).tolist() for n in (150, 160, 170)]
    outs = eng.generate(prompts, SamplingParams(temperature=0.0, max_tokens=60, ignore_eos=True))
    assert all(len(o.output_token_ids) == 60 for o in outs)
    assert eng.evictor.stats.sequences > 0 and eng.kv.num_free_blocks() == 40


def test_refusals_and_stats(tiny_cfg, tiny_weights):
    from fastapi.testclient import TestClient

    from gollek_b200.server.app import create_app
    from gollek_b200.server.async_engine import AsyncEngine
    ev = dict(kv_eviction=True, kv_eviction_policy="attention")
    for bad in (dict(kv_cache_dtype="auto", **ev), dict(kv_cache_dtype="fp8_block", kv_eviction=True), dict(block_size=8),
                dict(kv_eviction_policy="weights"), dict(speculative_method="ngram", **ev), dict(kv_cache_dtype="int4"),
                dict(tensor_parallel_size=2, **ev)):
        with pytest.raises(ValueError):
            engine(tiny_cfg, tiny_weights, **bad)
    eng = engine(tiny_cfg, tiny_weights)
    eng.generate([list(range(3, 60))], SamplingParams(temperature=0.0, max_tokens=2, ignore_eos=True))
    with pytest.raises(ValueError):
        eng.save_prefix_cache("/tmp/unused.safetensors")
    ae = AsyncEngine(engine(tiny_cfg, tiny_weights, **ev)).start()
    try:
        with TestClient(create_app(ae)) as c:
            assert c.get("/v1/kvcache/stats").json()["eviction_policy"] == "attention"
            assert c.post("/v1/kvcache/evict-now").json()["blocks_dropped"] == 0
    finally:
        ae.shutdown(drain=False)


@pytest.mark.parametrize("kind", ["int8", "fp8_block"])
@pytest.mark.parametrize("method", ["ngram", "draft"])
def test_speculation_is_refused(tiny_cfg, tiny_weights, kind, method):
    """A draft's row raises its block's scale and rounds the rows before it; a rejected draft leaves them so."""
    with pytest.raises(ValueError, match="coarsen"):
        engine(tiny_cfg, tiny_weights, kv_cache_dtype=kind, speculative_method=method)
    assert engine(tiny_cfg, tiny_weights, kv_cache_dtype="auto", speculative_method="ngram").spec is not None


def test_snapshot_of_another_cache_is_refused(tiny_cfg, tiny_weights, tmp_path):
    src = engine(tiny_cfg, tiny_weights, kv_cache_dtype="auto")
    src.generate([list(range(3, 100))], SamplingParams(temperature=0.0, max_tokens=2, ignore_eos=True))
    path = str(tmp_path / "prefix.safetensors")
    assert src.save_prefix_cache(path) > 0
    with pytest.raises(ValueError):
        engine(tiny_cfg, tiny_weights).load_prefix_cache(path)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,D", [("int8", 128), ("fp8_block", 128), ("int8", 64)])
def test_engine_tokens_gpu(kind, D):
    cfg = preset("llama-3-8b", num_hidden_layers=2, vocab_size=4096, head_dim=D)
    w = init_random_weights(cfg, seed=5)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 4096, (n,), generator=g).tolist() for n in (90, 17, 200)]
    eng = engine(cfg, w, device="cuda", kv_cache_dtype=kind, num_blocks=64)
    outs = eng.generate(prompts, SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True))
    for p, o in zip(prompts, outs):
        assert float(gaps(cfg, w, p, o.output_token_ids).max()) < 0.25


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
def test_decode_after_eviction_gpu(graphs):
    cfg = preset("llama-3-8b", num_hidden_layers=2, vocab_size=4096)
    w = init_random_weights(cfg, seed=6)
    eng, prompt, toks, gone, tokens, total = evicted_run(cfg, w, "cuda", use_cuda_graphs=graphs)
    check_evicted(cfg, w, prompt, toks, gone, tokens)


@pytest.mark.gpu
def test_captured_padding_rows_weigh_nothing_gpu():
    """Three sequences in a captured batch of four: the fourth row reads block 0, which may be somebody's."""
    cfg = preset("llama-3-8b", num_hidden_layers=1, vocab_size=4096)
    w = init_random_weights(cfg, seed=7)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 4096, (n,), generator=g).tolist() for n in (40, 20, 30)]
    eng = engine(cfg, w, device="cuda", num_blocks=32, kv_eviction=True, kv_eviction_policy="attention",
                 kv_eviction_threshold=1.1, async_scheduling=False)
    for i, p in enumerate(prompts):
        eng.add_request(str(i), p, SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True))
    steps = 0
    while all(len(s.output_token_ids) < 5 for s in eng.seqs.values()) and steps < 20:
        eng.step()
        steps += 1
    # every query that weighed added one softmax per head; a token's slot is zeroed when it is written
    torch.cuda.synchronize()
    total = float(eng.model.kv_mass.double().sum())
    queries = sum(len(s.output_token_ids) for s in eng.seqs.values())
    assert len(eng.seqs) == 3 and abs(total - queries * cfg.num_attention_heads) < 1e-2


@pytest.mark.parametrize("halves", [False, True])
def test_tables_are_as_wide_as_their_own_rows(tiny_cfg, tiny_weights, halves):
    """Decoding rows of 300 tokens beside prompts of 20 and the other way round: operators over an 8-bit cache size their
    copies and scores by the table, so neither call may get the step's widest row."""
    eng = engine(tiny_cfg, tiny_weights)
    if halves:
        eng.runner.split_min_tokens = 1
        eng.model.can_split_batch = lambda: True
    seen, forward = [], eng.model.forward

    def spy(ids, meta, cache, **kw):
        for m in meta.halves[1:] if meta.halves else (meta,):
            for kind in ("decode", "prefill"):
                bt, lens = getattr(m, kind + "_block_tables"), getattr(m, kind + "_seq_lens")
                if bt is not None and lens is not None and len(lens):
                    assert bt.shape[0] == len(lens)
                    seen.append((kind, bt.shape[1], max(1, -(-int(lens.max()) // 16)), m.num_decode > 0 and m.num_prefill_tokens > 0))
        meta.halves = None
        return forward(ids, meta, cache, **kw)

    eng.model.forward = spy
    g = torch.Generator().manual_seed(6)
    params = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)
    for at, n in ((0, 300), (2, 20), (3, 20), (6, 330)):
        while eng._steps < at:
            eng.step()
        eng.add_request(str(at), torch.randint(3, 250, (n,), generator=g).tolist(), params)
    while eng.has_unfinished():
        eng.step()
    assert {k for k, *_, mixed in seen if mixed} == {"decode", "prefill"} or halves
    assert all(w == need for _, w, need, _ in seen), seen
    assert any(w < 3 for _, w, *_ in seen) and any(w > 18 for _, w, *_ in seen)


@pytest.mark.gpu
def test_scores_are_held_before_the_pool_is_sized_gpu():
    """Weighing decode attention keeps a score for every head and token of the table's width: one buffer for all captured
    batches, allocated before the pool, and no captured batch brings one of its own."""
    cfg = preset("llama-3-8b", num_hidden_layers=1, vocab_size=4096)
    w = init_random_weights(cfg, seed=7)
    eng = engine(cfg, w, device="cuda", num_blocks=64, kv_eviction=True, kv_eviction_policy="attention", max_num_seqs=32,
                 max_model_len=32768, cuda_graph_batch_sizes=(8, 16, 32))
    scores = 32 * 32768 * cfg.num_attention_heads * 4
    assert eng.model.kv_workspace.numel() * 4 >= scores
    torch.cuda.synchronize()
    before = torch.cuda.memory_reserved()
    eng.runner.capture_all()
    assert len(eng.runner.graphs) == 3 and torch.cuda.memory_reserved() - before < scores
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 4096, (n,), generator=g).tolist() for n in (40, 20, 130)]
    outs = eng.generate(prompts, SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True))
    for p, o in zip(prompts, outs):
        assert float(gaps(cfg, w, p, o.output_token_ids).max()) < 0.25
