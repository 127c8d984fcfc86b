"""Beam search and the 8-bit cache through the engine on the GPU."""
import pytest
import torch

from coeus_b200.infer.engine import InferenceEngine
from coeus_b200.infer.scheduler import ContinuousBatcher
from coeus_b200.models.config import DecoderConfig
from coeus_b200.models.decoder import DecoderLM
from coeus_b200.ops import _lib
from coeus_b200.ops.ragged import Entry

pytestmark = pytest.mark.gpu
DEV = "cuda"


def model(kind):
    torch.manual_seed(0)
    kw = dict(hidden_dim=256, num_layers=2, num_heads=4, intermediate_dim=512, vocab_size=1000,
              max_seq_len=1024)
    if kind != "gpt":
        kw.update(use_bias=False, activation="swiglu", norm="rmsnorm", pos="rope")
    if kind == "gqa":
        kw.update(num_heads=2, num_kv_heads=1)
    return DecoderLM(DecoderConfig(**kw), device=DEV, training=False)


def status():
    torch.cuda.synchronize()
    return int(_lib.status_buffer(torch.device("cuda", 0))[0])


@pytest.mark.parametrize("kind", ["gpt", "llama", "gqa"])
@pytest.mark.parametrize("kv", [None, "int8", "e4m3"])
def test_beam_search(kind, kv):
    m = model(kind)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 1000, (3, 61), generator=g).to(DEV)
    n = 12
    eng = InferenceEngine(m, max_batch=12, kv_dtype=kv)
    out, scores = eng.beam_search(ids, 4, n, keep=4)
    again, s2 = InferenceEngine(m, max_batch=12, use_graph=False, kv_dtype=kv).beam_search(ids, 4, n, keep=4)
    assert torch.equal(out, again) and torch.equal(scores, s2)
    assert torch.equal(out[:, :, :61], ids[:, None].expand(3, 4, 61))
    assert all(len({tuple(x) for x in out[b].tolist()}) == 4 for b in range(3))
    # every sequence's score is what the whole model says of it: the logits, of size about 2, are
    # rounded to bf16 on both sides (2^-8 of it each), and so are a dozen intermediate results of a
    # layer; an 8-bit cache rounds keys and values by up to 2^-4 of them, averaged over the positions
    x = m.forward_logits(out.reshape(12, -1)[:, :-1])[..., :1000].float()
    lp = torch.log_softmax(x.view(12, -1, 1000), -1)[:, 60:]
    want = torch.gather(lp, 2, out.reshape(12, -1)[:, 61:, None])[..., 0].sum(-1).view(3, 4) / n
    assert float((want - scores).abs().max()) < (0.04 if kv is None else 0.08)
    one, _ = eng.beam_search(ids, 1, n)
    assert torch.equal(one[:, 0], eng.generate(ids, n))
    assert status() == 0


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
def test_8_bit_cache(kv):
    m = model("gqa")
    ids = torch.randint(0, 1000, (1, 200), generator=torch.Generator().manual_seed(2)).to(DEV)
    eng = InferenceEngine(m, max_batch=4, kv_dtype=kv)
    assert torch.equal(eng.generate(ids, 70), InferenceEngine(m, max_batch=4, kv_dtype=kv, use_graph=False).generate(ids, 70))
    eng.open_slots(4, 320)
    ref = InferenceEngine(m, max_batch=4)
    ref.open_slots(4, 320)
    for e in (eng, ref):
        e.prefill_slot(0, ids[0, :180], 256)
    got = eng.step([Entry(0, 180, ids[0, 180:].tolist(), list(range(20)))])
    want = ref.step([Entry(0, 180, ids[0, 180:].tolist(), list(range(20)))])
    size = float(want.float().abs().max())
    assert float((got.float() - want.float()).abs().max()) < 0.08 * size
    # on top of cached pages, and in chunks that read the earlier ones back
    a = eng.prefill_slot_paged(1, ids[0], 256, eng.cache.owned[0][:2])
    b = eng.prefill_slot(2, ids[0], 256, token_chunk=40)
    w = ref.prefill_slot(2, ids[0], 256)
    for x in (a, b):
        assert float((x.float() - w.float()).abs().max()) < 0.08 * size
    assert status() == 0


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
def test_batcher(kv):
    m = model("llama")
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (70, 3, 130, 64)]
    b = ContinuousBatcher(InferenceEngine(m, max_batch=4, kv_dtype=kv), max_seqs=3, max_len=256, prefix_cache=True)
    rids = [b.submit(p, 9) for p in prompts]
    out = b.run()
    assert all(len(out[r]) == 9 for r in rids)
    r = b.submit(prompts[2], 9)
    assert len(b.run()[r]) == 9 and b.prefix.hits == 1
    assert status() == 0


@pytest.mark.parametrize("kv", [None, "int8"])
def test_fewer_tokens_than_beams(kv):
    """The first step leaves places of the beam empty; scores are what the whole model says of the sequences, within
    the bounds of test_beam_search."""
    torch.manual_seed(0)
    m = DecoderLM(DecoderConfig(hidden_dim=256, num_layers=2, num_heads=4, intermediate_dim=512, vocab_size=3,
                                max_seq_len=256, use_bias=False, activation="swiglu", norm="rmsnorm", pos="rope"),
                  device=DEV, training=False)
    for S in (10, 64, 70):
        ids = torch.randint(0, 3, (2, S), generator=torch.Generator().manual_seed(S)).to(DEV)
        for graph in (True, False):
            out, scores = InferenceEngine(m, max_batch=16, use_graph=graph, kv_dtype=kv).beam_search(ids, 8, 6, keep=8)
            x = m.forward_logits(out.reshape(16, -1)[:, :-1])[..., :3].float()
            lp = torch.log_softmax(x.view(16, -1, 3), -1)[:, S - 1:]
            want = torch.gather(lp, 2, out.reshape(16, -1)[:, S:, None])[..., 0].sum(-1).view(2, 8) / 6
            assert float((want - scores).abs().max()) < (0.04 if kv is None else 0.08)
            assert all(len({tuple(x) for x in out[b].tolist()}) == 8 for b in range(2))
    assert status() == 0
