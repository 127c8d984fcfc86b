"""Beam search and the 8-bit cache through the engine, the batcher and the command line, on the CPU."""
import json
import math

import pytest
import torch

from coeus_b200.foundation.error import ProcessingError
from coeus_b200.infer.engine import InferenceEngine, make_engine
from coeus_b200.infer.scheduler import ContinuousBatcher
from coeus_b200.models.config import DecoderConfig
from coeus_b200.models.decoder import DecoderLM
from coeus_b200.ops.ragged import Entry


def model(kind="llama", vocab=61, seed=0):
    torch.manual_seed(seed)
    kw = dict(hidden_dim=128, num_layers=2, num_heads=2, intermediate_dim=192, vocab_size=vocab,
              max_seq_len=256)
    if kind != "gpt":
        kw.update(use_bias=False, activation="swiglu", norm="rmsnorm", pos="rope")
    if kind == "gqa":
        kw.update(num_heads=2, num_kv_heads=1)
    m = DecoderLM(DecoderConfig(**kw), device="cpu", dtype=torch.float32, training=False)
    for name, w in m.w.items():              # logits that are far from even
        if name.endswith("embed") or "output" in name:
            w.mul_(8.0)
    return m


def plain_beams(m, prompt, K, n, eos, penalty):
    """Beam search by recomputing the whole sequence of every beam for every token."""
    beams = [(0.0, [], False)]
    for _ in range(n):
        cand = []
        for j, (s, toks, over) in enumerate(beams):
            if over:
                cand.append((-s, j, eos, toks + [eos], True))
                continue
            ids = torch.tensor([prompt + toks])
            x = m.forward_logits(ids)[0, -1, :m.cfg.vocab_size].double()
            lp = torch.log_softmax(x, -1)
            top = torch.topk(lp, min(K, lp.numel()))
            for v, t in zip(top.values.tolist(), top.indices.tolist()):
                cand.append((-(s + v), j, t, toks + [t], t == eos))
        cand.sort(key=lambda c: c[:3])
        beams = [(-c[0], c[3], c[4]) for c in cand[:K]]
        if all(b[2] for b in beams):
            break
    out = []
    for s, toks, over in beams:
        c = toks.index(eos) + 1 if eos is not None and eos in toks else len(toks)
        out.append((s / c ** penalty, toks + [eos if eos is not None else 0] * (n - len(toks))))
    out.sort(key=lambda o: -o[0])
    return out


@pytest.mark.parametrize("kind", ["gpt", "llama", "gqa"])
@pytest.mark.parametrize("S,K,n,eos", [(5, 3, 6, None), (63, 4, 5, 7), (64, 2, 3, 7), (60, 1, 8, None)])
def test_beam_search_against_full_recomputation(kind, S, K, n, eos):
    m = model(kind)
    g = torch.Generator().manual_seed(S)
    ids = torch.randint(0, 61, (2, S), generator=g)
    out, scores = InferenceEngine(m, max_batch=8).beam_search(ids, K, n, eos_id=eos, length_penalty=0.7, keep=K)
    for b in range(2):
        want = plain_beams(m, ids[b].tolist(), K, n, eos, 0.7)
        for i in range(K):
            assert out[b, i, :S].tolist() == ids[b].tolist()
            assert out[b, i, S:].tolist() == want[i][1]
            # sums of fp32 log-probabilities of a few tokens
            assert abs(float(scores[b, i]) - want[i][0]) < 1e-4


def test_one_beam_is_greedy_and_a_beam_beyond_pages():
    m = model()
    eng = InferenceEngine(m, max_batch=8)
    ids = torch.randint(0, 61, (2, 50), generator=torch.Generator().manual_seed(1))
    greedy = eng.generate(ids, 90)
    out, _ = eng.beam_search(ids, 1, 90)
    assert torch.equal(out[:, 0], greedy)
    a, sa = eng.beam_search(ids, 4, 90, token_chunk=10)
    b, sb = eng.beam_search(ids[1:], 4, 90)
    assert torch.equal(a[1:], b) and torch.allclose(sa[1:], sb, atol=1e-4)
    assert bool((a[:, 0] != greedy).any())         # looking ahead finds something else here


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", ["gpt", "gqa"])
def test_engine_with_8_bit_cache(kv, kind):
    """One token at a time, several at once, on top of cached pages: the same numbers; and near those of
    the cache that is not rounded."""
    m = model(kind)
    ids = torch.randint(0, 61, (1, 150), generator=torch.Generator().manual_seed(2))
    eng = InferenceEngine(m, max_batch=4, kv_dtype=kv)
    eng.open_slots(4, 256)
    assert eng.cache.k[0].element_size() == 1
    eng.prefill_slot(0, ids[0, :140], 160)
    one = [eng.step([Entry(0, 140 + i, [int(ids[0, 140 + i])], [0])]) for i in range(10)]
    eng.prefill_slot(1, ids[0, :140], 160)
    many = eng.step([Entry(1, 140, ids[0, 140:].tolist(), list(range(10)))])
    # a chunk's tokens share the scale of their page from the start; with powers of two that only
    # moves where the smallest codes are rounded
    assert torch.allclose(torch.cat(one), many, atol=2e-2, rtol=0)
    pages = eng.cache.owned[0][:2]
    top = eng.prefill_slot_paged(2, ids[0], 160, pages)
    full = InferenceEngine(m, max_batch=4)
    full.open_slots(4, 256)
    want = full.prefill_slot(0, ids[0], 160)
    size = float(want.abs().max())
    for got in (many[-1], top):
        assert float((got - want).abs().max()) < 0.08 * size
    # chunks of a prompt read the earlier ones back
    eng.cache.release(3)
    a = eng.prefill_slot(3, ids[0], 160, token_chunk=50)
    assert float((a - want).abs().max()) < 0.08 * size


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
def test_batcher_and_beams_over_8_bits(kv):
    m = model("gqa")
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 61, (n,), generator=g).tolist() for n in (70, 3, 130)]
    alone = []
    for p in prompts:
        eng = InferenceEngine(m, max_batch=4, kv_dtype=kv)
        alone.append(eng.generate(torch.tensor([p]), 12)[0, len(p):].tolist())
    for prefix in (False, True):
        b = ContinuousBatcher(InferenceEngine(m, max_batch=4, kv_dtype=kv), max_seqs=2, max_len=256,
                              prefix_cache=prefix)
        rids = [b.submit(p, 12) for p in prompts]
        out = b.run()
        if not prefix:
            assert [out[r] for r in rids] == alone
        again = b.submit(prompts[2], 12)
        assert len(b.run()[again]) == 12
    eng = InferenceEngine(m, max_batch=8, kv_dtype=kv)
    one, _ = eng.beam_search(torch.tensor([prompts[0]]), 1, 12)
    assert one[0, 0, 70:].tolist() == alone[0]
    out, scores = eng.beam_search(torch.tensor([prompts[0]]), 4, 40, keep=4)
    assert out.shape == (1, 4, 110) and bool((scores[0, :-1] >= scores[0, 1:]).all())
    assert len({tuple(x) for x in out[0].tolist()}) == 4


def test_refusals():
    m = model()
    eng = InferenceEngine(m, max_batch=4)
    ids = torch.zeros((2, 5), dtype=torch.int64)
    for kw in (dict(beams=0), dict(beams=3), dict(beams=33), dict(beams=2, keep=3), dict(beams=2, max_new_tokens=0),
               dict(beams=2, eos_id=61)):
        with pytest.raises(ProcessingError):
            eng.beam_search(ids, **{"max_new_tokens": 3, **kw})
    with pytest.raises(ProcessingError):
        eng.beam_search(ids[:, :0], 2, 3)
    with pytest.raises(ProcessingError):
        InferenceEngine(m, kv_dtype="fp4")
    small = DecoderLM(DecoderConfig(hidden_dim=64, num_layers=1, num_heads=2, intermediate_dim=64,
                                    vocab_size=31, max_seq_len=64), device="cpu", training=False)
    with pytest.raises(ProcessingError):
        InferenceEngine(small, kv_dtype="int8")


def test_command_line(tmp_path, capsys):
    from coeus_b200.__main__ import main
    from coeus_b200.checkpoint.formats import save_model
    m = model("gpt")
    path = tmp_path / "m.safetensors"
    save_model(m, str(path))
    main(["generate", f"--weights={path}", "--prompt_ids=5,6,7", "--max_tokens=6", "--beams=3",
          "--kv_dtype=int8", "--device=cpu"])
    out = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert len(out["token_ids"]) == 6 and math.isfinite(out["score"]) and out["score"] < 0.0
    # one beam is the greedy continuation, which the end token ends too
    args = ["generate", f"--weights={path}", "--prompt_ids=5,6,7", "--max_tokens=6", "--device=cpu"]
    main(args)
    plain = json.loads(capsys.readouterr().out.strip().splitlines()[-1])["token_ids"]
    main(args + [f"--eos_id={plain[1]}"])
    ended = json.loads(capsys.readouterr().out.strip().splitlines()[-1])["token_ids"]
    first = plain.index(plain[1])
    assert ended[:first + 1] == plain[:first + 1] and set(ended[first + 1:]) <= {plain[1]}
    with pytest.raises(SystemExit):
        main(args + ["--beams=2", "--temperature=0.8"])


def test_mixed_layers_refuse_8_bits():
    from dogilorn_cases import Bench
    m = Bench("odd", "cpu", torch.float32).lm
    with pytest.raises(ProcessingError):
        make_engine(m, kv_dtype="int8")
    with pytest.raises(ProcessingError):
        make_engine(m).beam_search(torch.zeros((1, 3), dtype=torch.int64), 2, 3)


@pytest.mark.parametrize("V,K", [(3, 4), (5, 8), (7, 8), (2, 3)])
@pytest.mark.parametrize("S", [10, 63, 64])
def test_fewer_tokens_than_beams(V, K, S):
    """The first steps leave places of the beam empty; those beams' rows still name the prompt's last page."""
    for seed in range(3):
        m = model("gpt", vocab=V, seed=seed)
        ids = torch.randint(0, V, (1, S), generator=torch.Generator().manual_seed(seed))
        for eos in (None, 1):
            out, scores = InferenceEngine(m, max_batch=8).beam_search(ids, K, 5, eos_id=eos, keep=K)
            want = plain_beams(m, ids[0].tolist(), K, 5, eos, 1.0)
            for i, (score, tokens) in enumerate(want):
                assert abs(float(scores[0, i]) - score) < 1e-4
                assert out[0, i, S:].tolist() == tokens


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("pages", [0, 2])
def test_portions_behind_cached_pages(kv, pages):
    """The rest of a prompt goes through the layers in bounded portions, to the same cache and logits."""
    m = model("gqa")
    S = 250
    ids = torch.randint(0, 61, (S,), generator=torch.Generator().manual_seed(7))
    eng = InferenceEngine(m, max_batch=4, kv_dtype=kv)
    eng.open_slots(4, 320)
    eng.prefill_slot(0, ids, 260)
    cached = eng.cache.owned[0][:pages]
    rows = []
    through = eng._layers
    eng._layers = lambda x, *a, **kw: (rows.append(x.shape[0]), through(x, *a, **kw))[1]
    want = eng.prefill_slot_paged(1, ids, 260, cached)
    assert rows == [S - 64 * pages]
    kept = [[t[eng.cache.owned[1]].clone() for t in eng.cache.layer(l)] for l in range(2)]
    for chunk, most in ((64, 64), (100, 64), (128, 128), (30, 30)):
        rows.clear()
        got = eng.prefill_slot_paged(2, ids, 260, cached, token_chunk=chunk)
        assert max(rows) == min(most, S - 64 * pages) and sum(rows) == S - 64 * pages
        assert eng.cache.length(2) == S
        if chunk >= 64:                    # pages are written whole: the same codes, sums of fp32 in another order
            for l in range(2):
                for a, b in zip(kept[l], eng.cache.layer(l)):
                    b = b[eng.cache.owned[2]]
                    if a.dtype == torch.float32:
                        assert torch.equal(a, b)
                    else:
                        assert (a.view(torch.int8) != b.view(torch.int8)).float().mean() < 0.01
            assert float((got - want).abs().max()) < 0.02 * float(want.abs().max())
        else:                              # a page's scale may grow while it fills
            assert float((got - want).abs().max()) < 0.08 * float(want.abs().max())
        eng.cache.release(2)
    b = ContinuousBatcher(InferenceEngine(m, max_batch=4, kv_dtype=kv), max_seqs=2, max_len=300,
                          token_chunk=64, prefix_cache=True)
    through2 = b.engine._layers
    rows.clear()
    b.engine._layers = lambda x, *a, **kw: (rows.append(x.shape[0]), through2(x, *a, **kw))[1]
    rid = b.submit(ids.tolist(), 3)
    assert len(b.run()[rid]) == 3 and max(rows) == 64


def test_a_sequence_twice_in_a_step():
    m = model()
    eng = InferenceEngine(m, max_batch=4, kv_dtype="int8")
    eng.open_slots(4, 128)
    ids = torch.arange(20)
    for slot in (0, 1):
        eng.prefill_slot(slot, ids, 40)
    before = [t.clone() for l in range(2) for t in eng.cache.layer(l)]
    with pytest.raises(ProcessingError):
        eng.step([Entry(0, 20, [5], [0]), Entry(1, 20, [6], [0]), Entry(0, 21, [7], [0])])
    assert all(torch.equal(a, b) for a, b in zip(before, (t for l in range(2) for t in eng.cache.layer(l))))
    assert eng.step([Entry(0, 20, [5, 7], [1]), Entry(1, 20, [6], [0])]).shape[0] == 2


def test_length_penalty_goes_with_beams(tmp_path, capsys):
    from coeus_b200.__main__ import main
    from coeus_b200.checkpoint.formats import save_model
    path = tmp_path / "m.safetensors"
    save_model(model("gpt"), str(path))
    args = ["generate", f"--weights={path}", "--prompt_ids=5,6,7", "--max_tokens=4", "--device=cpu"]
    for more in (["--length_penalty=0.7"], ["--length_penalty=0.7", "--beams=1"]):
        with pytest.raises(SystemExit):
            main(args + more)
    capsys.readouterr()
    scores = []
    for penalty in ("1.0", "0.0"):
        main(args + ["--beams=2", f"--length_penalty={penalty}"])
        scores.append(json.loads(capsys.readouterr().out.strip().splitlines()[-1])["score"])
    assert abs(scores[0] * 4 - scores[1]) < 1e-5 * abs(scores[1])       # four tokens each: divided by 4, or by 1
